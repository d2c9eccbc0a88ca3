"""GPU parity of the 8-bit products at sizes that their tiles of 256 x 256 take: workgroups that go from tile to tile.

Whole numbers are exact through quantisation, products and sums (test_gpu_float8.py), so that results are the roundings of the products in 64 bits: equal
bits.  The products in 64 bits are made on the GPU.  Activations: oracle.float8_oracle.slack_of and the rounding, as there.
"""
from types import SimpleNamespace

import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F
from stk_amd.backend import _lib
from tests.test_gpu_float8 import DEV, _check, _n64, _route, _whole

pytestmark = pytest.mark.gpu
WIDE = 8   # stk_8bit_product_kernel


def _numbers(shape, seed, most=8):
    return torch.randint(-most, most + 1, shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=torch.int32)


def _product(a, b):
    return a.double() @ b.double()


# one block of inputs or several; tiles that fill the chip once, not quite and many times; rows, outputs and strides that are odd; half a tile of rows
SIZES = [(3500, 128, 3500), (5000, 100, 5000), (4097, 300, 4099), (9000, 640, 2306), (20000, 257, 8200), (70, 384, 49152), (66, 130, 50001), (300, 1153, 25000), (8192, 4096, 2048)]


@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_whole_numbers(rows, inputs, outputs):
    assert _lib.load().stk_8bit_product_kernel(rows, 1, inputs, outputs) == WIDE
    x, w = _numbers((rows, inputs), rows), _numbers((inputs, outputs), inputs)
    dtype = torch.float16 if rows % 3 == 0 else torch.bfloat16
    want = _product(x, w).float().to(dtype)
    assert torch.equal(stk.ops.matmul_8bit(x.to(dtype), stk.ops.quantize_8bit(w.to(dtype))), want)
    ones = torch.ones((inputs + 127) // 128, (outputs + 127) // 128, device=DEV)
    assert torch.equal(stk.ops.matmul_8bit(x.to(dtype), stk.ops.pack_8bit(w.to(torch.float8_e4m3fn), ones)), want)


@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", ["power", "float"])
def test_activations(activation, kind):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(80, 200, generator=g).bfloat16(), (torch.randn(200, 49160, generator=g) * 0.1).bfloat16()
    xq, wq = F.quantised(_n64(x), 1, 128)[0], F.quantised(_n64(w), 128, 128)[0]
    packed = stk.ops.quantize_8bit(w.to(DEV))
    if kind == "float":
        codes = torch.randint(-8, 9, (200, 49160), generator=g).float() / 8
        packed, wq = stk.ops.pack_8bit(codes.to(torch.float8_e4m3fn).to(DEV), torch.ones(2, 385, device=DEV)), _n64(codes)
    _check(stk.ops.matmul_8bit(x.to(DEV), packed, activation), xq @ wq, F.slack_of(xq, wq), torch.bfloat16, activation)


@pytest.mark.parametrize("tokens,experts,top_k,inputs,outputs,how", [(6000, 8, 2, 200, 1100, "any"), (4000, 16, 1, 130, 3000, "half"), (150000, 2100, 1, 24, 66, "any"),
                                                                      (3000, 6, 3, 257, 1539, "one"), (20000, 64, 1, 256, 770, "any")])
def test_routed(tokens, experts, top_k, inputs, outputs, how):
    assert _lib.load().stk_8bit_product_kernel(tokens * top_k, experts, inputs, outputs) == WIDE
    x, h, w = _numbers((tokens, inputs), 1), _numbers((tokens * top_k, inputs), 2), _numbers((experts, inputs, outputs), 3)
    if experts <= 1024:
        r = _route(tokens, experts, top_k, how, 1, tokens)
    else:   # (more than route makes)
        order = torch.sort(torch.randint(0, experts, (tokens * top_k,), device=DEV), stable=True)
        bins = torch.searchsorted(order.values, torch.arange(experts, device=DEV), right=True).int()
        r = SimpleNamespace(indices=order.indices.int(), bins=bins, top_k=top_k)
    packed = stk.ops.quantize_8bit(w.bfloat16())
    ends, slots = [0] + r.bins.tolist(), r.indices.long()
    sums, back = torch.empty(tokens * top_k, outputs, device=DEV), torch.empty(tokens * top_k, outputs, device=DEV)
    for e in range(experts):
        at = slots[ends[e]:ends[e + 1]]
        if at.numel():
            sums[ends[e]:ends[e + 1]] = _product(x[at // top_k], w[e]).float()
            back[at] = _product(h[ends[e]:ends[e + 1]], w[e]).float()
    assert torch.equal(stk.ops.gather_matmul_8bit(x.bfloat16(), r, packed, "relu"), sums.relu().bfloat16())
    by = 2.0 ** torch.randint(-2, 2, (tokens, top_k), device=DEV).float()
    want = (back.view(tokens, top_k, outputs).double() * by.double().unsqueeze(2)).sum(1)
    assert torch.equal(stk.ops.matmul_8bit_scatter(h.bfloat16(), r, packed, by), want.float().bfloat16())


@pytest.mark.parametrize("rows,inputs,outputs", [(3700, 3600, 3700), (130, 12800, 12810), (4100, 4097, 3585)])
def test_training_step(rows, inputs, outputs):
    x, w, grad = _numbers((rows, inputs), 1, 4), _numbers((inputs, outputs), 2, 4), _numbers((rows, outputs), 3, 2)
    a, b = x.bfloat16().requires_grad_(), w.bfloat16().requires_grad_()
    y = stk.ops.linear_8bit(a, b)
    dx, dw = torch.autograd.grad(y, (a, b), grad.bfloat16())
    for got, want in ((y, _product(x, w)), (dx, _product(grad, w.t().contiguous())), (dw, _product(x.t().contiguous(), grad))):
        assert torch.equal(got, want.float().bfloat16())


@pytest.mark.parametrize("tokens,experts,how,behind", [(9000, 8, "any", 0), (9000, 8, "half", 700), (2000, 40, "half", 128)])
def test_training_step_of_experts(tokens, experts, how, behind):
    inputs, outputs = 1300, 1290
    top = torch.randint(0, experts if how == "any" else experts // 2, (tokens, 1), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    need = int(stk.ops.route(top, experts, 128).padded_bins[-1])
    r = stk.ops.route(top, experts, 128, need + behind)
    rows, ends = need + behind, [0] + r.padded_bins.tolist()
    x, w, grad = _numbers((rows, inputs), 1, 4), _numbers((experts, inputs, outputs), 2, 4), _numbers((rows, outputs), 3, 2)
    a, b = x.half().requires_grad_(), w.half().requires_grad_()
    y = stk.ops.linear_8bit(a, b, r)
    dx, dw = torch.autograd.grad(y, (a, b), grad.half())
    for e in range(experts):
        at = slice(ends[e], ends[e + 1])
        assert torch.equal(y[at], _product(x[at], w[e]).float().half()), e
        assert torch.equal(dx[at], _product(grad[at], w[e].t().contiguous()).float().half()), e
        assert torch.equal(dw[e], _product(x[at].t().contiguous(), grad[at]).float().half()), e
    assert not y[need:].any() and not dx[need:].any()


def test_captured_and_on_two_streams():
    """Replays see new rows, and two calls under way at once have workspaces of their own."""
    w = stk.ops.quantize_8bit(_numbers((256, 4200), 1).bfloat16())
    x = _numbers((4000, 256), 2).bfloat16()
    stk.ops.matmul_8bit(x, w)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = stk.ops.matmul_8bit(x, w)
    for seed in range(3):
        x.copy_(_numbers((4000, 256), 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, stk.ops.matmul_8bit(x, w)), seed
    other = _numbers((4000, 256), 20).bfloat16()
    want = [stk.ops.matmul_8bit(t, w) for t in (x, other)]
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            there = stk.ops.matmul_8bit(other, w)
        here = stk.ops.matmul_8bit(x, w)
        torch.cuda.synchronize()
        assert torch.equal(here, want[0]) and torch.equal(there, want[1])
