"""GPU parity of every kernel of the products with 4-bit weights, with routing and without, at every class of groups, against the definition in
64 bits (computed on the device expert by expert).

Bounds as in test_gpu_weights4.py: sums are off by at most (inputs / 32 + 32) 2^-24 of the sum of |x| 32 |scale| plus |x offset|; on the way
back the top_k + 1 operations of a token's sum add 2^-24 of its terms' magnitudes each; a result is rounded once, to half a unit in the last place."""
import pytest
import torch

import stk_amd as stk
from tests._weights4_cases import GROUPS, KERNELS, PLAIN, ROUTED
from tests.test_gpu_weights4 import HALF, SMALL, _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _made(shape, group, affine, dtype, seed):
    codes, scales, offsets = (None if t is None else t.to(DEV) for t in _weights(shape, group, affine, dtype, seed))
    return codes, scales, offsets, stk.ops.pack_4bit(codes, scales, group, offsets)


def _exact(rows, codes, scales, offsets, group):
    """(sums, how far fp32 sums may be off) of rows and one matrix."""
    at = torch.arange(codes.size(0), device=DEV) // group
    s, c, x = scales.double()[at], codes.double(), rows.double()
    o = 0.0 if offsets is None else offsets.double()[at]
    w = s * (c - 8) if offsets is None else s * c + o
    slack = (codes.size(0) / 32 + 32) * 2.0 ** -24 * (x.abs() @ (32 * s.abs() + (o if offsets is None else o.abs())))
    return x @ w, slack


def _close(got, want, slack, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    bad = ~((got.double() - want).abs() <= 1.001 * HALF[dtype] * want.abs() + slack + SMALL[dtype])
    assert not bool(bad.any()), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())


FORMS = [(torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True), (torch.float16, False)]


@pytest.mark.parametrize("dtype,affine", FORMS)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("kernel", KERNELS)
def test_with_routing(kernel, group, dtype, affine):
    tokens, experts, top_k, inputs, outputs = ROUTED[kernel]
    codes, scales, offsets, w = _made((experts, inputs, outputs), group, affine, dtype, group + inputs)
    g = torch.Generator().manual_seed(tokens)
    # of unequal popularity; one expert without any where there are some to spare
    likely = torch.rand(experts, generator=g) + 0.1
    if experts > 2:
        likely[experts // 2] = 0.0
    top = torch.multinomial(likely.expand(tokens, experts), top_k, generator=g).to(torch.int32)
    route = stk.ops.route(top.to(DEV), experts, 1)
    x, h = torch.randn(tokens, inputs, generator=g).to(dtype).to(DEV), torch.randn(tokens * top_k, inputs, generator=g).to(dtype).to(DEV)
    by = (torch.rand(tokens, top_k, generator=g) + 0.1).to(DEV)
    there, back = stk.ops.gather_matmul_4bit(x, route, w), stk.ops.matmul_4bit_scatter(h, route, w, by)
    slots = route.indices.long()
    want = torch.zeros(tokens, outputs, dtype=torch.float64, device=DEV)
    slack, sizes, begin = torch.zeros_like(want), torch.zeros_like(want), 0
    assert int(route.bins[-1]) == tokens * top_k
    for e, end in enumerate(route.bins.tolist()):
        if end > begin:
            mine = slots[begin:end]
            matrix = (codes[e], scales[e], None if offsets is None else offsets[e], group)
            _close(there[begin:end], *_exact(x[mine // top_k], *matrix), dtype, ("there", e))
            sums, off = _exact(h[begin:end], *matrix)
            weight = by.view(-1)[mine].double().unsqueeze(1)
            # (a token is at an expert once)
            want[mine // top_k] += sums * weight
            slack[mine // top_k] += off * weight
            sizes[mine // top_k] += sums.abs() * weight
        begin = end
    _close(back, want, slack + (top_k + 1) * 2.0 ** -24 * sizes, dtype, "back")


@pytest.mark.parametrize("dtype,affine", FORMS[:2])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("kernel", KERNELS)
def test_without_routing(kernel, group, dtype, affine):
    rows, inputs, outputs = PLAIN[kernel]
    codes, scales, offsets, w = _made((inputs, outputs), group, affine, dtype, group + rows)
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).to(dtype).to(DEV)
    _close(stk.ops.matmul_4bit(x, w), *_exact(x, codes, scales, offsets, group), dtype, "plain")
