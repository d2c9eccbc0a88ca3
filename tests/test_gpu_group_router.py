"""GPU parity of the router's choice among groups of experts against the 64-bit definition.

Experts have to be equal, whatever fp32 makes of values that lie close together.  Weights: p is off by at most 2^-19 of itself in fp32 (an exponential of
two units in the last place, a sum of 1024 of them in a tree, a division), their sum and the division by it as much again, the rounding included: 2^-18.  A
gradient is a sum of two products of such factors: 2^-17 of the larger of them, then the rounding of its type.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# tokens, experts, groups, top_groups, top_k, best
CASES = [(1, 1, 1, 1, 1, 1), (5, 8, 1, 1, 2, 1), (64, 256, 8, 4, 8, 2), (33, 160, 8, 3, 6, 1), (100, 64, 16, 3, 4, 2), (17, 30, 3, 2, 10, 2), (7, 60, 60, 20, 16, 1),
         (9, 1024, 64, 5, 32, 2), (40, 1000, 8, 3, 17, 2), (50, 512, 16, 4, 16, 2), (3, 300, 1, 1, 8, 1), (200, 96, 2, 1, 12, 1), (11, 257, 1, 1, 32, 1), (130, 24, 4, 4, 24, 1)]


def _case(tokens, experts, dtype, seed, bias):
    g = torch.Generator().manual_seed(seed)
    scores = (torch.randn(tokens, experts, generator=g) * 1.5).to(dtype)
    return scores, torch.randn(experts, generator=g) * 0.1 if bias else None, g


def _check(scores, bias, top_k, groups, top_groups, best, scoring, normalize, scale, grad=None, what=""):
    s = scores.clone().to(DEV).requires_grad_(grad is not None)
    got, weights = stk.ops.group_top_experts(s, top_k, groups, top_groups, scoring, None if bias is None else bias.to(DEV), best, normalize, scale)
    n64 = scores.double().numpy()
    want, want_weights = F.group_choice(n64, top_k, groups, top_groups, scoring, None if bias is None else bias.double().numpy(), best, normalize, scale)
    assert got.dtype == torch.int32 and weights.dtype == torch.float32
    assert np.array_equal(got.cpu().numpy(), want), what
    off = np.abs(weights.detach().double().cpu().numpy() - want_weights)
    assert (off <= 2.0 ** -18 * np.abs(want_weights) + 2.0 ** -140).all(), (what, off.max())
    if grad is not None:
        ds, = torch.autograd.grad(weights, s, grad.to(DEV))
        exact = F.group_choice_gradient(n64, want, grad.double().numpy(), scoring, normalize, scale)
        u = np.abs(grad.double().numpy() * want_weights)
        size = np.zeros(n64.shape)
        np.put_along_axis(size, want, u, 1)
        p = np.zeros(n64.shape)
        if normalize:
            np.put_along_axis(p, want, np.abs(want_weights / scale), 1)
        elif scoring == "softmax":
            top = np.maximum(n64.max(1, keepdims=True), -1e300)     # (a row of masked experts: p is 0)
            p = np.exp(n64 - top) / np.maximum(np.exp(n64 - top).sum(1, keepdims=True), 1e-300)
        size = size + p * u.sum(1, keepdims=True)
        off = np.abs(ds.double().cpu().numpy() - exact)
        assert ds.dtype == scores.dtype and (off <= 2.0 ** -17 * size + HALF[scores.dtype] * np.abs(exact) + (2.0 ** -24 if scores.dtype == torch.float16 else 2.0 ** -126)).all(), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,normalize,bias", [("sigmoid", True, True), ("softmax", False, False), ("softmax", True, True), ("sigmoid", False, False), ("softmax", False, True)])
@pytest.mark.parametrize("tokens,experts,groups,top_groups,top_k,best", CASES)
def test_choice_and_gradient(tokens, experts, groups, top_groups, top_k, best, scoring, normalize, bias, dtype):
    scores, b, g = _case(tokens, experts, dtype, tokens + experts, bias)
    _check(scores, b, top_k, groups, top_groups, best, scoring, normalize, 2.5, torch.randn(tokens, top_k, generator=g))


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(64, 8, 4, 8), (256, 8, 4, 8), (500, 20, 5, 10)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_what_fp32_does_not_tell_apart(experts, groups, top_groups, top_k, scoring):
    """Biases that bring every c of a token to within some 1e-8 of one of three values, and group values with them."""
    g = torch.Generator().manual_seed(experts)
    s = torch.randn(1, experts, generator=g)
    n64 = s.double().numpy()[0]
    p = 1 / (1 + np.exp(-n64)) if scoring == "sigmoid" else np.exp(n64 - n64.max()) / np.exp(n64 - n64.max()).sum()
    level = torch.randint(1, 4, (experts,), generator=g).double().numpy() / 4
    bias = torch.from_numpy(level - p + 1e-8 * torch.randn(experts, generator=g).double().numpy()).float()
    _check(s.repeat(70, 1), bias, top_k, groups, top_groups, 2, scoring, True, 1.0)
    _check(s.repeat(3, 1), bias, top_k, 1, 1, 1, scoring, False, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "zero", "some"])
def test_ties(dtype, scoring, bias):
    """Scores of few values: equal inputs go to the lower number."""
    g = torch.Generator().manual_seed(3)
    s = torch.randint(-2, 3, (200, 128), generator=g).to(dtype)
    b = None if bias is None else torch.zeros(128) if bias == "zero" else torch.randint(0, 3, (128,), generator=g) * 0.25
    for groups, top_groups, best in ((1, 1, 1), (8, 3, 1), (8, 3, 2)):
        _check(s, b, 9, groups, top_groups, best, scoring, True, 1.0)
        _check(torch.zeros(5, 128, dtype=dtype), b, 9, groups, top_groups, best, scoring, True, 1.0)


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("bias", [False, True])
def test_masks(scoring, normalize, bias):
    """Experts masked by -infinity: single ones, all but a few (fewer than are chosen), whole groups, the whole row; and the type's lowest value."""
    scores, b, g = _case(60, 64, torch.float32, 1, bias)
    scores[torch.rand(60, 64, generator=g) < 0.5] = -float("inf")
    scores[0, 3:] = -float("inf")
    scores[1] = -float("inf")
    scores[2, :32] = -float("inf")
    scores[3, ::2] = torch.finfo(torch.float32).min
    scores[4, 1:] = torch.finfo(torch.float32).min
    grad = torch.randn(60, 8, generator=g)
    for groups, top_groups, best in ((1, 1, 1), (8, 4, 2), (8, 2, 1)):
        _check(scores, b, 8, groups, top_groups, best, scoring, normalize, 1.0, grad, (groups, best))


def test_saturated_scores():
    """Sigmoids that are 1 or 0 to the last bit keep the order of their scores where there is no bias."""
    s = torch.linspace(-200, 200, 96)[torch.randperm(96, generator=torch.Generator().manual_seed(2))].repeat(4, 1)
    _check(s, None, 20, 1, 1, 1, "sigmoid", False, 1.0, torch.ones(4, 20))
    _check(s, None, 20, 1, 1, 1, "softmax", False, 1.0, torch.ones(4, 20))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_are_not_numbers(scoring, bad):
    scores, b, _ = _case(20, 64, torch.float32, 5, True)
    want, want_weights = stk.ops.group_top_experts(scores.to(DEV), 6, 8, 3, scoring, b.to(DEV))
    scores[::3, 17] = bad
    got, weights = stk.ops.group_top_experts(scores.to(DEV), 6, 8, 3, scoring, b.to(DEV))
    keep = [t for t in range(20) if t % 3]
    assert torch.equal(got[keep], want[keep]) and torch.equal(weights[keep], want_weights[keep])
    assert all(len(set(row)) == 6 and 0 <= min(row) and max(row) < 64 for row in got.cpu().tolist())
    if not (scoring == "sigmoid" and bad > 0):
        assert weights[::3].isnan().all() if scoring == "softmax" else weights[::3].isnan().any()
    for extreme in (float("inf"), -float("inf"), float("nan")):
        wild = b.clone()
        wild[9] = extreme
        got, weights = stk.ops.group_top_experts(scores[keep].to(DEV), 6, 8, 3, scoring, wild.to(DEV))
        assert torch.isfinite(weights).all() and bool((got == 9).any(1).all()) == (extreme != -float("inf"))


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_differences(scoring, normalize):
    """The gradient against differences of the 64-bit definition: the choice stays where it is over so short a way, and what is cut off is of the order of 1e-10."""
    scores, b, g = _case(6, 48, torch.float32, 11, True)
    grad, way = torch.randn(6, 5, generator=g), torch.randn(6, 48, generator=g).double().numpy()
    s = scores.to(DEV).requires_grad_()
    _, weights = stk.ops.group_top_experts(s, 5, 4, 2, scoring, b.to(DEV), 2, normalize, 2.0)
    ds, = torch.autograd.grad(weights, s, grad.to(DEV))
    f = lambda h: (F.group_choice(scores.double().numpy() + h * way, 5, 4, 2, scoring, b.double().numpy(), 2, normalize, 2.0)[1] * grad.double().numpy()).sum()
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs((ds.double().cpu().numpy() * way).sum() - want) <= 1e-4 * max(1.0, abs(want))


def test_strides_streams_and_empty():
    scores, b, g = _case(50, 64, torch.bfloat16, 4, True)
    want = stk.ops.group_top_experts(scores.to(DEV), 4, 8, 2, "sigmoid", b.to(DEV))
    wide = torch.zeros(50, 80, dtype=torch.bfloat16, device=DEV)
    wide[:, 7:71] = scores.to(DEV)
    turned = scores.t().contiguous().to(DEV).t()
    for view in (wide[:, 7:71], turned):
        got = stk.ops.group_top_experts(view, 4, 8, 2, "sigmoid", b.to(DEV))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = stk.ops.group_top_experts(wide[:, 7:71], 4, 8, 2, "sigmoid", b.to(DEV))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    none = torch.empty(0, 64, device=DEV, requires_grad=True)
    chosen, weights = stk.ops.group_top_experts(none, 4, 8, 2)
    assert chosen.shape == weights.shape == (0, 4) and torch.autograd.grad(weights.sum(), none)[0].shape == (0, 64)


def test_refusals():
    s = torch.zeros(4, 64, device=DEV)
    ok = dict(top_k=4, groups=8, top_groups=2)
    for wrong in (dict(top_k=0), dict(top_k=17), dict(groups=7), dict(groups=0), dict(top_groups=9), dict(top_groups=0), dict(group_best=3), dict(group_best=0),
                  dict(groups=64, top_groups=8), dict(bias=torch.zeros(63, device=DEV)), dict(scale=0.0), dict(scale=float("inf"))):
        with pytest.raises(AssertionError):
            stk.ops.group_top_experts(s, **{**ok, **wrong})
    for wrong in (s.double(), s.to(torch.int32), torch.zeros(4, 1025, device=DEV)):
        with pytest.raises(NotImplementedError):
            stk.ops.group_top_experts(wrong, 2)
    with pytest.raises(NotImplementedError):
        stk.ops.group_top_experts(torch.zeros(4, 80, device=DEV), 33)
    with pytest.raises(RuntimeError):
        stk.ops.group_top_experts(s, 2, bias=torch.zeros(64))
    with pytest.raises(AssertionError):
        stk.ops.group_top_experts(s[0], 2)


# more tokens than get a wavefront each
MANY = [(2100, 256, 8, 4, 8, 2), (3000, 160, 8, 3, 6, 1), (2500, 64, 16, 3, 4, 2), (2049, 30, 3, 2, 10, 2), (4001, 8, 1, 1, 2, 1), (2300, 128, 2, 1, 16, 1), (2200, 100, 1, 1, 5, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring,normalize,bias", [("sigmoid", True, True), ("softmax", False, False), ("softmax", True, True), ("sigmoid", False, False)])
@pytest.mark.parametrize("tokens,experts,groups,top_groups,top_k,best", MANY)
def test_many_tokens(tokens, experts, groups, top_groups, top_k, best, scoring, normalize, bias, dtype):
    scores, b, g = _case(tokens, experts, dtype, tokens + experts, bias)
    _check(scores, b, top_k, groups, top_groups, best, scoring, normalize, 2.5, torch.randn(tokens, top_k, generator=g))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_many_tokens_that_fp32_does_not_tell_apart(scoring):
    """Some of the tokens of a workgroup, or all."""
    g = torch.Generator().manual_seed(8)
    s = torch.randn(1, 256, generator=g)
    n64 = s.double().numpy()[0]
    p = 1 / (1 + np.exp(-n64)) if scoring == "sigmoid" else np.exp(n64 - n64.max()) / np.exp(n64 - n64.max()).sum()
    level = torch.randint(1, 4, (256,), generator=g).double().numpy() / 4
    bias = torch.from_numpy(level - p + 1e-8 * torch.randn(256, generator=g).double().numpy()).float()
    scores = s.repeat(2100, 1)
    scores[1000:] += (torch.rand(1100, 1, generator=g) < 0.7) * torch.randn(1100, 256, generator=g)
    _check(scores, bias, 8, 8, 4, 2, scoring, True, 1.0)
    _check(scores, bias, 8, 1, 1, 1, scoring, False, 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "some"])
def test_many_tokens_of_ties_and_masks(scoring, bias):
    g = torch.Generator().manual_seed(3)
    s = torch.randint(-2, 3, (2200, 128), generator=g).float()
    s[500:1500][torch.rand(1000, 128, generator=g) < 0.5] = -float("inf")
    s[700], s[701, 3:], s[702, :64], s[703, 1:] = -float("inf"), -float("inf"), -float("inf"), torch.finfo(torch.float32).min
    b = None if bias is None else torch.randint(0, 3, (128,), generator=g) * 0.25
    grad = torch.randn(2200, 9, generator=g)
    for groups, top_groups, best in ((1, 1, 1), (8, 3, 1), (8, 3, 2)):
        _check(s, b, 9, groups, top_groups, best, scoring, True, 1.0, grad, (groups, best))
    s[::7, 17] = float("nan")
    got, weights = stk.ops.group_top_experts(s.to(DEV), 9, 8, 3, scoring, None if b is None else b.to(DEV))
    assert all(len(set(row)) == 9 and 0 <= min(row) and max(row) < 128 for row in got[::7].cpu().tolist()) and weights[::7].isnan().any(1).any()
