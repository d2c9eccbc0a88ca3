"""GPU parity of stk.ops.top_experts and its gradient against the 64-bit definition.

The choice is exact.  Weights are fp32: score - largest is off by 2^-24 of its size, so that exp of it is off by that in relative terms, and
the function, the sum of at most 1024 terms and the quotient add a few units each: (64 + spread) 2^-24, spread the largest |score - largest|
that still counts (beyond 104 exp is 0 in fp32).  A gradient is a difference of two such terms, rounded once to the scores' type.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import layer_oracle as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = 2.0 ** -120
SIZES = [(1, 1, 1), (5, 2, 1), (7, 3, 3), (64, 64, 2), (1000, 8, 2), (33, 27, 5), (300, 256, 8), (50, 129, 4), (9, 1024, 64), (4, 1000, 1), (257, 64, 1),
         (20, 16, 16), (11, 513, 7), (3, 65, 64), (130, 4, 4)]


def _n64(t):
    return t.detach().double().cpu().numpy()


def _check(scores, top_k, normalize, grad, chosen, weights, dscores):
    s = _n64(scores)
    want_chosen, want = L.top_experts(s, top_k, normalize)
    assert chosen.dtype == torch.int32 and weights.dtype == torch.float32
    assert np.array_equal(chosen.cpu().numpy(), want_chosen)
    eps = (64 + 104) * 2.0 ** -24
    got = _n64(weights)
    assert (np.abs(got - want) <= eps * want + TINY).all(), np.abs(got - want).max()
    if dscores is None:
        return
    want = L.top_experts_gradient(s, top_k, _n64(grad), normalize)
    terms = (np.abs(_n64(grad)) * got).sum(axis=1, keepdims=True)
    own = np.zeros(s.shape)
    np.put_along_axis(own, want_chosen, np.abs(_n64(grad)) * got, axis=1)
    assert dscores.dtype == scores.dtype
    small = 2.0 ** -24 if scores.dtype == torch.float16 else TINY
    bad = ~(np.abs(_n64(dscores) - want) <= HALF[scores.dtype] * np.abs(want) * 1.001 + 2 * eps * (own + terms) + small)
    assert not bad.any(), (np.argwhere(bad)[0], _n64(dscores)[bad][0], want[bad][0])


def _run(scores, top_k, normalize, grad):
    leaf = scores.detach().requires_grad_(True)
    chosen, weights = stk.ops.top_experts(leaf, top_k, normalize)
    assert not chosen.requires_grad
    d, = torch.autograd.grad(weights, leaf, grad)
    return chosen, weights.detach(), d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k", SIZES)
def test_choice_weights_and_gradient(tokens, experts, top_k, normalize, dtype):
    g = torch.Generator().manual_seed(tokens + experts)
    scores = (torch.randn(tokens, experts, generator=g) * 3).to(dtype).to(DEV)
    grad = torch.randn(tokens, top_k, generator=g).to(DEV)
    chosen, weights, d = _run(scores, top_k, normalize, grad)
    _check(scores, top_k, normalize, grad, chosen, weights, d)
    with torch.no_grad():
        again = stk.ops.top_experts(scores, top_k, normalize)
    assert torch.equal(again[0], chosen) and torch.equal(again[1], weights)


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (64, 4), (200, 8), (1024, 3)])
def test_ties_go_to_the_lower_expert(experts, top_k, normalize):
    g = torch.Generator().manual_seed(experts)
    scores = torch.randint(-2, 2, (100, experts), generator=g).float()
    scores[scores == 0] = torch.where(torch.rand(int((scores == 0).sum()), generator=g) < 0.5, 0.0, -0.0)
    scores[0] = 1.5
    grad = torch.randn(100, top_k, generator=g).to(DEV)
    scores = scores.to(DEV)
    _check(scores, top_k, normalize, grad, *_run(scores, top_k, normalize, grad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("experts,top_k", [(6, 3), (64, 4), (100, 2)])
def test_masked_experts(experts, top_k, normalize, dtype):
    g = torch.Generator().manual_seed(experts)
    scores = torch.randn(40, experts, generator=g)
    scores[torch.rand(40, experts, generator=g) < 0.6] = -float("inf")
    scores[3], scores[4] = -float("inf"), -float("inf")          # rows that the mask leaves empty
    scores[4, experts - 1] = 0.5                                 # one expert left, the others fill the places
    scores[5] = torch.finfo(dtype).min                           # the lowest value is a number: all alike
    scores[6] = torch.finfo(dtype).min
    scores[6, 2] = torch.finfo(dtype).max                        # as far apart as the type allows
    scores = scores.to(dtype).to(DEV)
    grad = torch.randn(40, top_k, generator=g).to(DEV)
    chosen, weights, d = _run(scores, top_k, normalize, grad)
    _check(scores, top_k, normalize, grad, chosen, weights, d)
    assert not weights[3].any() and not d[3].any() and chosen[3].tolist() == list(range(top_k))
    assert weights[4].tolist() == [1.0] + [0.0] * (top_k - 1)


def test_nan_and_infinity_stay_in_their_rows():
    scores = torch.randn(6, 20, generator=torch.Generator().manual_seed(4))
    scores[1, 7], scores[1, 3], scores[4, 9] = float("nan"), float("nan"), float("inf")
    scores = scores.to(DEV)
    grad = torch.ones(6, 2, device=DEV)
    for normalize in (False, True):
        chosen, weights, d = _run(scores, 2, normalize, grad)
        assert chosen[1].tolist() == [3, 7] and int(chosen[4, 0]) == 9
        rest = [0, 2, 3, 5]
        _check(scores[rest], 2, normalize, grad[rest], chosen[rest], weights[rest], d[rest])
        assert torch.isnan(weights[[1, 4]]).all()
        assert torch.isnan(d[[1, 4]]).any(dim=1).all()
        assert 0 <= int(chosen.min()) and int(chosen.max()) < 20


@pytest.mark.parametrize("normalize", [False, True])
def test_strides(normalize):
    g = torch.Generator().manual_seed(6)
    scores, grad = torch.randn(30, 17, generator=g), torch.randn(30, 3, generator=g).to(DEV)
    want = _run(scores.to(DEV), 3, normalize, grad)
    wide = torch.full((30, 40), 9.0, device=DEV)
    wide[:, 5:22] = scores.to(DEV)
    for view in (wide[:, 5:22], scores.t().contiguous().to(DEV).t(), torch.stack([scores, scores], dim=2).to(DEV)[:, :, 1]):
        got = _run(view, 3, normalize, grad)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one row of scores for every token, one gradient for every weight
    row = scores.to(DEV)[:1].expand(30, 17)
    got = stk.ops.top_experts(row, 3, normalize)
    assert torch.equal(got[0], want[0][:1].expand(30, 3)) and torch.equal(got[1], want[1][:1].expand(30, 3))
    leaf = scores.to(DEV).requires_grad_(True)
    a, = torch.autograd.grad(stk.ops.top_experts(leaf, 3, normalize)[1].sum(), leaf)
    assert torch.equal(a, _run(leaf, 3, normalize, torch.ones(30, 3, device=DEV))[2])


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(7)
    scores, grad = torch.randn(4, 6, generator=g), torch.randn(4, 2, generator=g)
    for normalize in (False, True):
        _, _, d = _run(scores.to(DEV), 2, normalize, grad.to(DEV))
        f = lambda s: (L.top_experts(s, 2, normalize)[1] * _n64(grad)).sum()
        for at in np.ndindex(4, 6):
            step = np.zeros((4, 6))
            step[at] = 1e-6
            assert abs((f(_n64(scores) + step) - f(_n64(scores) - step)) / 2e-6 - float(d[at])) < 1e-6


def test_feeds_the_routing():
    g = torch.Generator().manual_seed(8)
    scores = torch.randn(200, 16, generator=g).to(DEV)
    chosen, weights = stk.ops.top_experts(scores, 2, normalize=True)
    route = stk.ops.route(chosen, 16, 128)
    x = torch.randn(200, 64, generator=g).to(DEV).bfloat16()
    back = stk.ops.padded_scatter(stk.ops.padded_gather(x, route), route, weights)
    # weights add up to 1: the rows come back, one rounding to bfloat16 later
    assert (back.float() - x.float()).abs().max() <= 2.0 ** -7 * x.float().abs().max()


def test_streams_and_graphs():
    g = torch.Generator().manual_seed(9)
    scores, grad = torch.randn(3000, 64, generator=g).to(DEV), torch.randn(3000, 2, generator=g).to(DEV)
    want = _run(scores, 2, False, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(scores, 2, False, grad)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = _run(scores, 2, False, grad)
    for replay in range(3):
        scores.copy_(torch.randn(scores.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, _run(scores, 2, False, grad))), replay


def test_no_tokens():
    chosen, weights, d = _run(torch.empty(0, 8, device=DEV), 2, False, torch.empty(0, 2, device=DEV))
    assert chosen.shape == weights.shape == (0, 2) and d.shape == (0, 8)


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for call in (lambda: stk.ops.top_experts(x, 9), lambda: stk.ops.top_experts(x, 0), lambda: stk.ops.top_experts(x.view(2, 2, 8), 1)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: stk.ops.top_experts(x.double(), 2), lambda: stk.ops.top_experts(torch.zeros(2, 1025, device=DEV), 2),
                 lambda: stk.ops.top_experts(torch.zeros(2, 100, device=DEV), 65)):
        with pytest.raises(NotImplementedError):
            call()
    leaf = torch.randn(4, 8, device=DEV, requires_grad=True)
    first, = torch.autograd.grad(stk.ops.top_experts(leaf, 2)[1].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: stk.ops.top_experts(s, 2)[1])(x.view(2, 2, 8))


def test_a_traced_call_computes_its_result_again():
    x = torch.randn(6, 12, generator=torch.Generator().manual_seed(1)).to(DEV)
    traced = torch.jit.trace(lambda v: stk.ops.top_experts(v, 2)[1], (x,), check_trace=False)
    assert torch.equal(traced(x.flip(0)), stk.ops.top_experts(x.flip(0), 2)[1])
