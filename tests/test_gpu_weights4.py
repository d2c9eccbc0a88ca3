"""GPU parity of the 4-bit weights and their products against the 64-bit definition.

Formats are exact.  A product's sums are fp32 in an order of the kernel's own: off by at most (inputs / 32 + 32) 2^-24 of the sum of
|x| 32 |scale| (the codes are multiplied as numbers up to 31, what is too much is taken off as sums of x) plus |x offset|; the
activations' slopes stay below 1.2, their own errors below 2^-20; the result is rounded once, to half a unit in the last place.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import layer_oracle as L
from stk_amd.backend import hip_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def _n64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _weights(shape, group, affine, dtype, seed):
    """(codes, scales, offsets), on the host."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8)
    groups = (*shape[:-2], (shape[-2] + group - 1) // group, shape[-1])
    scales = ((torch.rand(groups, generator=g) + 0.2) * 0.05).to(dtype)
    return codes, scales, (torch.randn(groups, generator=g) * 0.2).to(dtype) if affine else None


def _pack(codes, scales, offsets, group):
    return stk.ops.pack_4bit(codes.to(DEV), scales.to(DEV), group, None if offsets is None else offsets.to(DEV))


def _slack(x, codes, scales, offsets, group):
    """[rows, outputs] for one matrix."""
    rows = np.arange(codes.shape[0]) // group
    size = 32 * np.abs(_n64(scales))[rows] + (0 if offsets is None else np.abs(_n64(offsets))[rows])
    return (codes.shape[0] / 32 + 32) * 2.0 ** -24 * (np.abs(_n64(x)) @ size)


ACT = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"),
       "silu": torch.nn.functional.silu}


def _check(got, sums, slack, dtype, activation=None, what=""):
    want = ACT[activation](torch.from_numpy(np.ascontiguousarray(sums))).numpy()
    assert got.dtype == dtype and tuple(got.shape) == want.shape, what
    if activation:
        slack = 1.2 * slack + 2.0 ** -20 * np.abs(sums)
    bad = ~(np.abs(_n64(got) - want) <= 1.001 * HALF[dtype] * np.abs(want) + slack + SMALL[dtype])
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[0].tolist(), _n64(got)[bad][0], want[bad][0])


# ---------------------------------------------------------------------------------------------------- formats
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("shape,group", [((1, 1), 32), ((128, 16), 128), ((129, 17), 64), ((300, 50), 32), ((3, 257, 33), 256), ((2, 64, 100), 128), ((5, 96, 16), 32)])
def test_packed_weights_come_back(shape, group, affine, dtype):
    codes, scales, offsets = _weights(shape, group, affine, dtype, sum(shape))
    w = _pack(codes, scales, offsets, group)
    assert (w.inputs, w.outputs, w.group_size, w.experts) == (*shape[-2:], group, shape[0] if len(shape) == 3 else None)
    got = stk.ops.dequantize_4bit(w)
    # 4 times 8 or 11 bits fit into fp32, and so does the sum but for its one rounding
    rows = torch.arange(shape[-2]) // group
    s = scales.float()[..., rows, :]
    want = s * (codes.float() - 8) if offsets is None else s * codes.float() + offsets.float()[..., rows, :]
    assert got.dtype == dtype and torch.equal(got.cpu(), want.to(dtype))


def test_codes_of_any_strides_and_high_bits():
    codes, scales, _ = _weights((64, 48), 32, False, torch.bfloat16, 3)
    want = stk.ops.dequantize_4bit(_pack(codes, scales, None, 32))
    turned = stk.ops.pack_4bit(codes.to(DEV).t().contiguous().t(), scales.to(DEV).t().contiguous().t(), 32)
    assert torch.equal(stk.ops.dequantize_4bit(turned), want)
    assert torch.equal(stk.ops.dequantize_4bit(_pack(codes | 0xf0, scales, None, 32)), want)


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.bfloat16, None), (torch.float16, None), (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("shape,group", [((256, 96), 128), ((100, 33), 32), ((4, 130, 20), 64), ((70, 5), 256)])
def test_quantized_weights_are_the_nearest(shape, group, affine, dtype, scale_dtype):
    g = torch.Generator().manual_seed(sum(shape))
    w = (torch.randn(shape, generator=g) * 0.1 + 0.02).to(dtype)
    w[..., 1:2] = 0.0                                            # an output without weights
    q = stk.ops.quantize_4bit(w.to(DEV), group, offsets=affine, dtype=scale_dtype)
    to = scale_dtype or dtype
    got = _n64(stk.ops.dequantize_4bit(q))
    rows = np.arange(shape[-2]) // group
    wn = _n64(w)
    for k in range(rows.max() + 1):
        part = wn[..., rows == k, :]
        if affine:
            scale = (part.max(axis=-2) - part.min(axis=-2)) / 15
            reach = 0.5 * scale + (16 * scale + np.abs(part.min(axis=-2))) * HALF[to]   # half a step, and the rounding of scale and offset
        else:
            scale = np.abs(part).max(axis=-2) / 7
            reach = 0.5 * scale + 8 * scale * HALF[to]
        err = np.abs(got[..., rows == k, :] - part).max(axis=-2)
        bound = reach * (1 + 2 * HALF[to]) + np.abs(part).max(axis=-2) * HALF[to] + 2 * SMALL[to]
        assert (err <= bound).all(), (err - bound).max()


def test_quantizes_views_of_the_layers_weights():
    g = torch.Generator().manual_seed(5)
    w1 = torch.randn(64, 4 * 32, generator=g).bfloat16().to(DEV)              # [hidden, experts * ffn]
    view = w1.view(64, 4, 32).transpose(0, 1)
    a, b = stk.ops.quantize_4bit(view, 32), stk.ops.quantize_4bit(view.contiguous(), 32)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)
    t = view.contiguous().transpose(1, 2).contiguous().transpose(1, 2)       # one row per output
    assert torch.equal(stk.ops.quantize_4bit(t, 32).packed, b.packed)


# ---------------------------------------------------------------------------------------------------- products
SIZES = [(1, 1, 1, 32), (1, 128, 16, 128), (1, 4096, 256, 128), (2, 8, 15, 32), (5, 200, 16, 64), (16, 1152, 100, 32), (17, 31, 33, 32), (33, 512, 64, 512),
         (64, 1024, 200, 128), (100, 300, 1151, 64), (257, 640, 80, 256), (3, 129, 17, 128), (130, 1000, 48, 64), (7, 2944, 128, 32), (48, 384, 400, 384),
         (600, 256, 272, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs,group", SIZES)
def test_product(rows, inputs, outputs, group, affine, dtype):
    codes, scales, offsets = _weights((inputs, outputs), group, affine, dtype, rows + inputs)
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).to(dtype)
    w = _pack(codes, scales, offsets, group)
    sums, slack = _n64(x) @ L.weights4(codes.numpy(), _n64(scales), group, _n64(offsets)), _slack(x, codes, scales, offsets, group)
    got = stk.ops.matmul_4bit(x.to(DEV), w)
    _check(got, sums, slack, dtype)
    assert torch.equal(got, stk.ops.matmul_4bit(x.to(DEV), w))
    activation = list(ACT)[1 + (rows + inputs) % 4]
    _check(stk.ops.matmul_4bit(x.to(DEV), w, activation), sums, slack, dtype, activation)


# one size for every kernel that the launch rule chooses from; inputs of no multiple of eight take the way through registers
BY_RULE = [(2100, 392, 2050, 128), (2100, 395, 2050, 32), (530, 264, 2048, 64), (530, 257, 2048, 128), (200, 136, 2050, 32), (200, 3080, 2050, 128), (550, 3080, 2050, 64),
           (40, 520, 2050, 128), (9, 300, 12001, 64), (3, 3080, 11000, 128), (3300, 264, 2050, 128)]


@pytest.mark.parametrize("dtype,affine", [(torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("rows,inputs,outputs,group", BY_RULE)
def test_product_of_every_kernel(rows, inputs, outputs, group, affine, dtype):
    codes, scales, offsets = _weights((inputs, outputs), group, affine, dtype, rows + inputs)
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).to(dtype)
    got = stk.ops.matmul_4bit(x.to(DEV), _pack(codes, scales, offsets, group))
    _check(got, _n64(x) @ L.weights4(codes.numpy(), _n64(scales), group, _n64(offsets)), _slack(x, codes, scales, offsets, group), dtype)


@pytest.mark.parametrize("rows", [40, 300])
def test_rows_of_a_view_give_the_same(rows):
    """Rows that lie in whole 16-byte pieces and rows that do not: another kernel, sums in the same order."""
    codes, scales, _ = _weights((264, 2064), 128, False, torch.bfloat16, 11)
    w = _pack(codes, scales, None, 128)
    x = torch.randn(rows, 264, generator=torch.Generator().manual_seed(rows)).bfloat16().to(DEV)
    off = torch.empty(rows * 264 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(rows, 264).copy_(x)
    assert torch.equal(stk.ops.matmul_4bit(off, w), stk.ops.matmul_4bit(x, w))


@pytest.mark.parametrize("activation", list(ACT))
def test_activations(activation):
    codes, scales, _ = _weights((256, 64), 128, False, torch.bfloat16, 1)
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).bfloat16() * 3
    got = stk.ops.matmul_4bit(x.to(DEV), _pack(codes, scales, None, 128), activation)
    _check(got, _n64(x) @ L.weights4(codes.numpy(), _n64(scales), 128), _slack(x, codes, scales, None, 128), torch.bfloat16, activation)


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
@pytest.mark.parametrize("inputs", [64, 333, 1024])
def test_strides_of_the_rows(rows, inputs):
    dtype = torch.float16
    codes, scales, _ = _weights((inputs, 70), 64, False, dtype, 2)
    w = _pack(codes, scales, None, 64)
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).to(dtype).to(DEV)
    want = stk.ops.matmul_4bit(x, w)
    wide = torch.full((rows, inputs + 9), float("nan"), dtype=dtype, device=DEV)
    off = torch.full((rows * inputs + 1,), float("nan"), dtype=dtype, device=DEV)[1:].view(rows, inputs)
    for view in (wide[:, 8:8 + inputs], wide[:, 3:3 + inputs], off, torch.empty(inputs, rows, dtype=dtype, device=DEV).t(),
                 torch.empty(rows, 2 * inputs, dtype=dtype, device=DEV)[:, ::2]):
        view.copy_(x)
        assert torch.equal(stk.ops.matmul_4bit(view, w), want)
    assert torch.equal(stk.ops.matmul_4bit(x[:1].expand(rows, inputs), w), want[:1].expand(rows, 70))
    assert torch.equal(stk.ops.matmul_4bit(x.view(1, rows, inputs), w), want.view(1, rows, 70))


def _route(tokens, experts, top_k, how, blocking, seed):
    g = torch.Generator().manual_seed(seed)
    if how == "one":
        top = torch.full((tokens, top_k), experts - 1, dtype=torch.int32)    # everything to the last expert
    elif how == "half":
        top = torch.randint(0, experts, (tokens, top_k), generator=g, dtype=torch.int32)
        top[: tokens // 2] = experts // 2
    else:
        top = torch.rand(tokens, experts, generator=g).topk(top_k, dim=1).indices.to(torch.int32)
    rows = None if blocking == 1 else stk.ops.route_capacity(tokens * top_k, experts, blocking)
    return stk.ops.route(top.to(DEV), experts, blocking, padded_rows=rows)


ROUTED = [(1, 4, 1, 128, 16, 128, "any", 1), (1, 64, 2, 256, 48, 64, "any", 128), (3, 4, 4, 200, 33, 32, "any", 1), (64, 64, 2, 256, 64, 128, "any", 1),
          (100, 8, 2, 384, 100, 128, "half", 1), (50, 200, 1, 64, 16, 64, "any", 1), (300, 4, 1, 130, 40, 32, "one", 1), (33, 16, 3, 512, 80, 256, "any", 64),
          (500, 6, 2, 256, 96, 128, "half", 1), (17, 1, 1, 128, 20, 128, "any", 1), (40, 32, 8, 96, 24, 32, "any", 1), (5, 1024, 2, 32, 16, 32, "any", 1),
          (2000, 3, 1, 160, 144, 32, "any", 128), (160, 64, 2, 136, 1120, 128, "any", 1), (600, 16, 2, 264, 528, 64, "half", 1), (1000, 8, 2, 264, 1040, 32, "half", 1),
          (300, 8, 2, 137, 1040, 128, "any", 1), (2, 4, 2, 3200, 700, 64, "any", 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k,inputs,outputs,group,how,blocking", ROUTED)
def test_routed_products(tokens, experts, top_k, inputs, outputs, group, how, blocking, affine, dtype):
    codes, scales, offsets = _weights((experts, inputs, outputs), group, affine, dtype, tokens + experts)
    w = _pack(codes, scales, offsets, group)
    r = _route(tokens, experts, top_k, how, blocking, tokens)
    g = torch.Generator().manual_seed(tokens)
    slots = tokens * top_k
    x, h, by = torch.randn(tokens, inputs, generator=g).to(dtype), torch.randn(slots, inputs, generator=g).to(dtype), torch.rand(tokens, top_k, generator=g) + 0.1
    indices, bins = r.indices.cpu().numpy(), r.bins.cpu().numpy()
    wn = L.weights4(codes.numpy(), _n64(scales), group, _n64(offsets))
    expert = np.searchsorted(bins, np.arange(slots), side="right")
    slack_of = lambda rows: np.concatenate([_slack(rows[p:p + 1], codes[e], scales[e], None if offsets is None else offsets[e], group) for p, e in enumerate(expert)])
    got = stk.ops.gather_matmul_4bit(x.to(DEV), r, w, "silu")
    _check(got, L.gather_matmul(_n64(x), indices, bins, top_k, wn), slack_of(x[torch.from_numpy(indices // top_k).long()]), dtype, "silu", "gather")
    assert torch.equal(got, stk.ops.gather_matmul_4bit(x.to(DEV), r, w, "silu"))
    for weights in (by, None):
        got = stk.ops.matmul_4bit_scatter(h.to(DEV), r, w, None if weights is None else weights.to(DEV))
        bn = np.ones(slots) if weights is None else _n64(weights).reshape(-1)
        slack, each, sizes = np.zeros((tokens, outputs)), slack_of(h), np.zeros((tokens, outputs))
        for p, s in enumerate(indices):
            slack[s // top_k] += each[p] * bn[s]
            sizes[s // top_k] += np.abs(_n64(h)[p] @ wn[expert[p]]) * bn[s]
        _check(got, L.matmul_scatter(_n64(h), indices, bins, top_k, wn, None if weights is None else bn), slack + (top_k + 1) * 2.0 ** -24 * sizes, dtype, None, "scatter")
        assert torch.equal(got, stk.ops.matmul_4bit_scatter(h.to(DEV), r, w, None if weights is None else weights.to(DEV)))


def test_experts_without_rows_are_not_read():
    """Scales of NaN in experts that no token is sent to."""
    codes, scales, _ = _weights((8, 128, 32), 128, False, torch.bfloat16, 4)
    scales[[0, 2, 3, 7]] = float("nan")   # (their codes' numbers and scales would make NaN of whatever they met)
    w = _pack(codes, scales, None, 128)
    top = torch.tensor([[1, 4], [5, 6], [6, 1]], dtype=torch.int32, device=DEV)
    r = stk.ops.route(top, 8, 1)
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    h = stk.ops.gather_matmul_4bit(x, r, w)
    assert torch.isfinite(h).all()
    assert torch.isfinite(stk.ops.matmul_4bit_scatter(x.repeat(2, 1), r, w)).all()


def test_no_rows():
    codes, scales, _ = _weights((4, 128, 32), 128, False, torch.bfloat16, 4)
    w = _pack(codes, scales, None, 128)
    r = stk.ops.route(torch.zeros(0, 2, dtype=torch.int32, device=DEV), 4, 1)
    assert stk.ops.gather_matmul_4bit(torch.empty(0, 128, device=DEV, dtype=torch.bfloat16), r, w).shape == (0, 32)
    assert stk.ops.matmul_4bit_scatter(torch.empty(0, 128, device=DEV, dtype=torch.bfloat16), r, w).shape == (0, 32)
    one = _pack(codes[0], scales[0], None, 128)
    assert stk.ops.matmul_4bit(torch.empty(0, 128, device=DEV, dtype=torch.bfloat16), one).shape == (0, 32)


def test_streams_and_graphs():
    codes, scales, _ = _weights((8, 512, 256), 128, False, torch.bfloat16, 6)
    back = _weights((8, 256, 512), 64, True, torch.bfloat16, 7)
    w1, w2 = _pack(codes, scales, None, 128), _pack(*back, 64)
    g = torch.Generator().manual_seed(3)
    x, top, by = torch.randn(40, 512, generator=g).bfloat16().to(DEV), torch.randint(0, 8, (40, 2), generator=g, dtype=torch.int32).to(DEV), torch.rand(40, 2, generator=g).to(DEV)

    def layer():
        r = stk.ops.route(top, 8, 1, padded_rows=80)
        return stk.ops.matmul_4bit_scatter(stk.ops.gather_matmul_4bit(x, r, w1, "gelu"), r, w2, by)

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = layer()
    for replay in range(3):
        x.copy_(torch.randn(x.shape, generator=g)), top.copy_(torch.randint(0, 8, top.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, layer()), replay


def test_refusals():
    codes, scales, offsets = _weights((128, 32), 64, True, torch.bfloat16, 8)
    w = _pack(codes, scales, offsets, 64)
    experts = stk.ops.quantize_4bit(torch.zeros(4, 128, 32, dtype=torch.bfloat16, device=DEV))
    x = torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV)
    r = stk.ops.route(torch.zeros(3, 1, dtype=torch.int32, device=DEV), 4, 1)
    other = stk.ops.route(torch.zeros(3, 1, dtype=torch.int32, device=DEV), 5, 1)
    c, s, o = codes.to(DEV), scales.to(DEV), offsets.to(DEV)
    for call in (lambda: stk.ops.matmul_4bit(x[:, :127], w), lambda: stk.ops.matmul_4bit(x, experts), lambda: stk.ops.gather_matmul_4bit(x, r, w),
                 lambda: stk.ops.gather_matmul_4bit(x[:2], r, experts), lambda: stk.ops.gather_matmul_4bit(x, other, experts),
                 lambda: stk.ops.matmul_4bit_scatter(x[:2], r, experts), lambda: stk.ops.matmul_4bit_scatter(x, r, experts, torch.ones(4, 1, device=DEV)),
                 lambda: stk.ops.pack_4bit(c, s[:1], 64), lambda: stk.ops.pack_4bit(c, s, 64, o[:, :31]), lambda: stk.ops.pack_4bit(c, s, 128),
                 lambda: stk.ops.matmul_4bit(x, w._replace(outputs=64)), lambda: stk.ops.pack_4bit(c, s, 64, o.half())):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: stk.ops.matmul_4bit(x.half(), w), lambda: stk.ops.matmul_4bit(x.float(), w), lambda: stk.ops.pack_4bit(c.int(), s, 64),
                 lambda: stk.ops.pack_4bit(c, s.float(), 64), lambda: stk.ops.quantize_4bit(torch.zeros(96, 4, device=DEV, dtype=torch.half), 48),
                 lambda: stk.ops.quantize_4bit(torch.zeros(96, 4, device=DEV)), lambda: stk.ops.matmul_4bit(x.clone().requires_grad_(True), w)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(ValueError):
        stk.ops.matmul_4bit(x, w, "gelu_grad")
    with pytest.raises(RuntimeError):
        stk.ops.matmul_4bit(x.cpu(), w)
    with pytest.raises(RuntimeError):
        stk.ops.matmul_4bit_scatter(x, r, experts, torch.ones(3, 1))
    assert hip_kernels.matmul_4bit(x, *w[:3], *w[4:]).shape == (3, 32)


@pytest.mark.parametrize("rows,outputs", [(2, 40), (20, 40), (100, 40), (100, 4100), (700, 1100)])
def test_infinite_and_nan_rows(rows, outputs):
    """They are NaN throughout, whatever the weights, and leave the other rows alone."""
    for dtype in HALF:
        codes, scales, offsets = _weights((300, outputs), 32, True, dtype, 9)
        x = torch.randn(rows, 300, generator=torch.Generator().manual_seed(rows)).to(dtype).to(DEV)
        for w in (_pack(codes, scales, None, 32), _pack(codes, scales, offsets, 32)):
            want = stk.ops.matmul_4bit(x, w)
            bad = x.clone()
            bad[1, 299] = float("inf")
            bad[rows - 1, 5] = float("nan")
            got = stk.ops.matmul_4bit(bad, w)
            for r in range(rows):
                assert torch.isnan(got[r]).all() if r in (1, rows - 1) else torch.equal(got[r], want[r])


def test_values_behind_the_last_input_are_not_used():
    """Rows of 100 inputs in storage that holds NaN right behind each of them."""
    codes, scales, _ = _weights((100, 2000), 64, False, torch.bfloat16, 10)
    w = _pack(codes, scales, None, 64)
    for rows in (1, 30, 90, 300):
        wide = torch.full((rows, 104), float("nan"), dtype=torch.bfloat16, device=DEV)
        wide[:, :100] = torch.randn(rows, 100, generator=torch.Generator().manual_seed(rows)).to(DEV)
        assert torch.equal(stk.ops.matmul_4bit(wide[:, :100], w), stk.ops.matmul_4bit(wide[:, :100].contiguous(), w))
        assert torch.isfinite(stk.ops.matmul_4bit(wide[:, :100], w)).all()


def test_autocast_and_inference_mode():
    """Under autocast rows of another type are cast like those of the other products; without it they are refused."""
    codes, scales, _ = _weights((2, 128, 48), 64, False, torch.bfloat16, 12)
    w = _pack(codes, scales, None, 64)
    one = _pack(codes[0], scales[0], None, 64)
    x = torch.randn(6, 128, generator=torch.Generator().manual_seed(13)).to(DEV)
    r = stk.ops.route(torch.tensor([0, 1, 1, 0, 1, 0], dtype=torch.int32, device=DEV).view(6, 1), 2, 1)
    back = _pack(codes.transpose(1, 2).contiguous(), scales[:, :1, :1].expand(2, 1, 128).contiguous(), None, 64)
    near = x.bfloat16()
    for layer in (lambda x: stk.ops.matmul_4bit(x, one), lambda x: stk.ops.matmul_4bit_scatter(stk.ops.gather_matmul_4bit(x, r, w), r, back)):
        want = layer(near)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(layer(x), want)
        with torch.inference_mode():
            assert torch.equal(layer(near), want)
        with pytest.raises(NotImplementedError):
            layer(x)
