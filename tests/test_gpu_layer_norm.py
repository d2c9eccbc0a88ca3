"""GPU parity of stk.ops.layer_norm and its gradients against the 64-bit definition.

Bounds.  A result is rounded once: half a unit in the last place of its type, U = 2^-8 (bfloat16), 2^-11 (float16), 2^-24 (float32) of its
own size.  Before that it is an fp32 computation: x - mean is off by up to 2^-24 of the largest |x| in each of a few
steps, and sums of n values by up to (n / 256 + 16) 2^-24 of the sum of their magnitudes (at most n / 256 values one after the other
in a thread, then a tree).  In units of the deviation that is E = (n / 256 + 16) 2^-24 (1 + max |x| / deviation) on a
normalised value, which weights and gradients multiply.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import layer_oracle as L
from stk_amd.backend import hip_kernels
from tests import _util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}   # (below it the spacing is fixed)
SIZES = [(1, 1), (3, 2), (5, 7), (64, 1024), (17, 1151), (9, 4100), (2, 20000), (300, 64), (1000, 80), (4099, 1152), (7, 8192), (1, 40000), (3000, 16), (33, 2049)]


def _inputs(rows, size, dtype, param, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, size, generator=g) * (torch.rand(size, generator=g) + 0.5) + offset).to(dtype)
    w, b = (1 + 0.3 * torch.randn(size, generator=g)).to(param), (0.3 * torch.randn(size, generator=g)).to(param)
    return x, w, b, torch.randn(rows, size, generator=g).to(dtype)


def _n64(t):
    return t.detach().double().cpu().numpy()


def _check(got, want, dtype, slack, what):
    got = _n64(got)
    assert got.shape == want.shape, what
    bound = HALF[dtype] * np.abs(want) + slack + SMALLEST[dtype]
    bad = ~(np.abs(got - want) <= bound * 1.001)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[0].tolist(), got[bad][0], want[bad][0], np.broadcast_to(bound, bad.shape)[bad][0])


def _check_all(y, grads, x, w, b, dy, eps=1e-5):
    """y and (dx, dw, db) of a call, on whatever device, against the definition."""
    xn, wn, bn, gn = _n64(x), None if w is None else _n64(w), None if b is None else _n64(b), _n64(dy)
    n = xn.shape[1]
    want, z, r = L.layer_norm(xn, wn, bn, eps)
    e = (n / 256 + 16) * 2.0 ** -24 * (1 + np.abs(xn).max(axis=1, keepdims=True) * r)
    big_w = 1.0 if wn is None else np.abs(wn)
    _check(y, want, y.dtype, e * (1 + np.abs(z)) * big_w + 2.0 ** -24 * (0 if bn is None else np.abs(bn)), "y")
    if grads is None:
        return
    dx, dw, db = L.layer_norm_gradients(gn, xn, wn, eps)
    g = np.abs(gn * big_w)
    # each of the three terms of dx is off by E times the largest of what it is made of
    _check(grads[0], dx, grads[0].dtype, r * e * (1 + np.abs(z)) * (2 * g + 2 * g.max(axis=1, keepdims=True) * (1 + np.abs(z).max(axis=1, keepdims=True))), "dx")
    steps = (len(xn) / 128 + 128) * 2.0 ** -24    # sums over rows: shares of the rows one by one, then the shares
    if w is not None:
        _check(grads[1], dw, grads[1].dtype, (np.abs(gn) * (e * (1 + np.abs(z)) + steps * np.abs(z))).sum(axis=0), "dw")
    if b is not None:
        _check(grads[2], db, grads[2].dtype, steps * np.abs(gn).sum(axis=0), "db")


def _run(x, w, b, dy, eps=1e-5):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = stk.ops.layer_norm(x, w, b, eps)
    found = list(torch.autograd.grad(y, leaves, dy))
    for t in leaves:
        t.requires_grad_(False)
    return y.detach(), [found.pop(0) if t is not None else None for t in (x, w, b)]


@pytest.mark.parametrize("dtype,param", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                         (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,size", SIZES)
def test_forward_and_gradients(rows, size, dtype, param):
    x, w, b, dy = (t.to(DEV) for t in _inputs(rows, size, dtype, param, rows + size))
    y, grads = _run(x, w, b, dy)
    assert y.dtype == grads[0].dtype == dtype and grads[1].dtype == grads[2].dtype == param
    _check_all(y, grads, x, w, b, dy)
    # without gradients the same bits, and again the same gradients
    with torch.no_grad():
        assert torch.equal(stk.ops.layer_norm(x, w, b), y)
    for a, c in zip(_run(x, w, b, dy)[1], grads):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_weight,with_bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("size", [37, 1024])
def test_without_parameters(size, with_weight, with_bias, dtype):
    x, w, b, dy = (t.to(DEV) for t in _inputs(40, size, dtype, dtype, size))
    w, b = w if with_weight else None, b if with_bias else None
    y, grads = _run(x, w, b, dy)
    _check_all(y, grads, x, w, b, dy)


@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)])
def test_any_of_the_gradients(wanted):
    x, w, b, dy = (t.to(DEV) for t in _inputs(50, 200, torch.float32, torch.float32, 5))
    _, whole = _run(x, w, b, dy)
    leaves = (x, w, b)
    for t, want in zip(leaves, wanted):
        t.requires_grad_(want)
    got = torch.autograd.grad(stk.ops.layer_norm(x, w, b), [t for t, want in zip(leaves, wanted) if want], dy)
    for a, c in zip(got, [c for c, want in zip(whole, wanted) if want]):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,eps", [(100.0, 1e-5), (0.0, 1.0), (-3.0, 0.0)])
def test_large_means_and_other_eps(offset, eps, dtype):
    x, w, b, dy = (t.to(DEV) for t in _inputs(30, 1000, dtype, dtype, 8, offset))
    y, grads = _run(x, w, b, dy, eps)
    _check_all(y, grads, x, w, b, dy, eps)


def test_constant_rows_have_no_deviation():
    x = torch.full((4, 100), 3.0, device=DEV, dtype=torch.bfloat16)
    w, b = torch.full((100,), 2.0, device=DEV, dtype=torch.bfloat16), torch.full((100,), 0.25, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(stk.ops.layer_norm(x, w, b), torch.full_like(x, 0.25))


def test_infinite_and_nan_values_stay_in_their_rows():
    x, w, b, dy = (t.to(DEV) for t in _inputs(6, 300, torch.float32, torch.float32, 9))
    clean, _ = _run(x, w, b, dy)
    x[1, 7], x[3, 0] = float("inf"), float("nan")
    y, grads = _run(x, w, b, dy)
    for row in range(6):
        if row in (1, 3):
            assert torch.isnan(y[row]).all() and torch.isnan(grads[0][row]).all()
        else:
            assert torch.equal(y[row], clean[row]) and torch.isfinite(grads[0][row]).all()


STRIDES = {
    "rows further apart": lambda x: torch.cat([x, x], dim=1)[:, :x.size(1)],
    "odd distance, odd start": lambda x: torch.empty(x.size(0) * (x.size(1) + 3) + 1, dtype=x.dtype)[1:].view(x.size(0), -1)[:, :x.size(1)],
    "every second value": lambda x: torch.empty(x.size(0), 2 * x.size(1), dtype=x.dtype)[:, ::2],
    "transposed": lambda x: torch.empty(x.size(1), x.size(0), dtype=x.dtype).t(),
}


@pytest.mark.parametrize("size", [64, 1023])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", list(STRIDES))
def test_strides(name, dtype, size):
    x, w, b, dy = _inputs(21, size, dtype, dtype, 11)
    xs, ds = STRIDES[name](x.to(DEV).cpu()), STRIDES[name](dy)
    xs.copy_(x), ds.copy_(dy)
    # (the views are made again on the device, where a copy would be contiguous)
    on = lambda like, v: torch.empty_strided(like.shape, like.stride(), dtype=like.dtype, device=DEV).copy_(v)
    y, grads = _run(on(xs, x), w.to(DEV), b.to(DEV), on(ds, dy))
    _check_all(y, grads, x, w, b, dy)
    again, other = _run(x.to(DEV), w.to(DEV), b.to(DEV), dy.to(DEV))
    assert torch.equal(y, again) and torch.equal(grads[0], other[0])


def test_a_start_off_the_16_byte_grid():
    x, w, b, dy = _inputs(21, 64, torch.bfloat16, torch.bfloat16, 12)
    off = lambda v: torch.empty(v.numel() + 1, dtype=v.dtype, device=DEV)[1:].view(v.shape).copy_(v)
    y, grads = _run(off(x), off(w), off(b), off(dy))
    _check_all(y, grads, x, w, b, dy)


def test_leading_dimensions_and_broadcast_rows():
    x, w, b, dy = (t.to(DEV) for t in _inputs(24, 48, torch.float32, torch.float32, 13))
    want, grads = _run(x, w, b, dy)
    for shape in [(2, 3, 4, 48), (24, 1, 48), (1, 24, 48)]:
        y, g = _run(x.view(shape).clone(), w, b, dy.view(shape))
        assert y.shape == shape and torch.equal(y.view(24, 48), want) and torch.equal(g[0].view(24, 48), grads[0]) and torch.equal(g[1], grads[1])
    y, g = _run(x.view(4, 6, 48).transpose(0, 1), w, b, dy.view(4, 6, 48).transpose(0, 1))
    assert torch.equal(y.transpose(0, 1).reshape(24, 48), want) and torch.equal(g[0].transpose(0, 1).reshape(24, 48), grads[0])
    assert torch.equal(stk.ops.layer_norm(x[0], w, b), want[0])
    # one row for all, and the gradient of a sum, which is one value for all
    row = x[:1].expand(5, 48)
    assert torch.equal(stk.ops.layer_norm(row, w, b), want[:1].expand(5, 48))
    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(stk.ops.layer_norm(leaf, w, b).sum(), leaf)
    assert torch.equal(got, _run(x, w, b, torch.ones_like(dy))[1][0])


def test_no_rows():
    w, b = torch.ones(32, device=DEV), torch.ones(32, device=DEV)
    y, grads = _run(torch.empty(0, 32, device=DEV), w, b, torch.empty(0, 32, device=DEV))
    assert y.shape == (0, 32) and grads[0].shape == (0, 32)
    assert not grads[1].any() and not grads[2].any()


def test_gradient_against_differences():
    x, w, b, dy = _inputs(3, 19, torch.float32, torch.float32, 14)
    _, grads = _run(x.to(DEV), w.to(DEV), b.to(DEV), dy.to(DEV))
    f = lambda x, w, b: (L.layer_norm(x, w, b)[0] * _n64(dy)).sum()
    h = 1e-6
    for k, t in enumerate((x, w, b)):
        for at in np.ndindex(*t.shape):
            values = [_n64(v) for v in (x, w, b)]
            step = np.zeros(t.shape)
            step[at] = h
            up, down = list(values), list(values)
            up[k], down[k] = values[k] + step, values[k] - step
            # differences: h^2 times a third derivative of a few units; fp32: a few 2^-24 of sums of 19 to 57 values
            assert abs((f(*up) - f(*down)) / (2 * h) - float(grads[k][at])) < 1e-5, (k, at)


def test_a_tensor_of_another_stream():
    x, w, b, dy = (t.to(DEV) for t in _inputs(512, 1024, torch.bfloat16, torch.bfloat16, 15))
    want, grads = _run(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, g = _run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want) and all(torch.equal(a, c) for a, c in zip(g, grads))


def test_replays_from_a_graph():
    x, w, b, dy = (t.to(DEV) for t in _inputs(700, 1024, torch.bfloat16, torch.bfloat16, 16))
    _run(x, w, b, dy)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, g = _run(x, w, b, dy)
    for replay in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(replay)))
        graph.replay()
        torch.cuda.synchronize()
        want, grads = _run(x, w, b, dy)
        assert torch.equal(y, want) and all(torch.equal(a, c) for a, c in zip(g, grads)), replay


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(AssertionError):
        stk.ops.layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(AssertionError):
        stk.ops.layer_norm(x.half(), torch.ones(8, device=DEV).half(), torch.ones(8, device=DEV))
    with pytest.raises(NotImplementedError):
        stk.ops.layer_norm(x, None, torch.ones(8, device=DEV).half())
    with pytest.raises(NotImplementedError):
        stk.ops.layer_norm(x, torch.ones(8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError):
        stk.ops.layer_norm(x.double())
    with pytest.raises(AssertionError):
        stk.ops.layer_norm(torch.zeros(4, 0, device=DEV))
    with pytest.raises(RuntimeError):
        stk.ops.layer_norm(x, torch.ones(8))
    # a gradient of the gradient, forward-mode differentiation and transforms are refused, not answered wrongly
    leaf = torch.randn(4, 8, device=DEV, requires_grad=True)
    first, = torch.autograd.grad(stk.ops.layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()
    with pytest.raises(RuntimeError):
        torch.func.vmap(stk.ops.layer_norm)(x.view(2, 2, 8))
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        stk.ops.layer_norm(forward_ad.make_dual(x, torch.ones_like(x)))


def test_statistics_are_those_of_the_rows():
    x, w, b, _ = _inputs(12, 500, torch.float16, torch.float16, 17)
    _, statistics = hip_kernels.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5, with_statistics=True)
    _, _, r = L.layer_norm(U.np32(x))
    np.testing.assert_allclose(_n64(statistics[0]), U.np32(x).astype(np.float64).mean(axis=1), rtol=0, atol=20 * 2.0 ** -24 * float(x.float().abs().max()))
    np.testing.assert_allclose(_n64(statistics[1]), r[:, 0], rtol=40 * 2.0 ** -24)


def test_a_traced_call_computes_its_result_again():
    x, w, b, _ = (t.to(DEV) for t in _inputs(5, 64, torch.float32, torch.float32, 18))
    traced = torch.jit.trace(lambda v: stk.ops.layer_norm(v, w, b), (x,), check_trace=False)
    other = x.flip(0) * 2
    assert torch.equal(traced(other), stk.ops.layer_norm(other, w, b))
