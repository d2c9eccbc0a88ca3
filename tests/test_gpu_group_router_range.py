"""A router's choice among groups at the ends of the range: sigmoids and softmaxes that fp32 has no number for.

Weights are held to the definition in logarithms, in 64 bits: log p of a sigmoid is s - log(1 + exp(s)), of a softmax s - log sum exp, and a normalised weight is
scale exp(log p - log sum exp(log p of the chosen)).  As in test_gpu_group_router.py they may be off by 2^-18 of themselves; beside it by the smallest step of fp32.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2.0 ** -149


def _log_sum(v):
    top = v.max(1, keepdims=True)
    return top + np.log(np.exp(v - top).sum(1, keepdims=True))


def _weights(scores, chosen, scoring, normalize, scale):
    log_p = scores - (np.logaddexp(0.0, scores) if scoring == "sigmoid" else _log_sum(scores))
    log_p = np.take_along_axis(log_p, chosen, 1)
    return scale * np.exp(log_p - (_log_sum(log_p) if normalize else 0.0))


def _check(scores, bias, scoring, normalize, scale, groups=1, top_groups=1, top_k=6):
    """scores: float32 on the host; the gradient against the oracle's."""
    grad = torch.randn(scores.shape[0], top_k, generator=torch.Generator().manual_seed(1))
    s = scores.to(DEV).requires_grad_()
    chosen, weights = stk.ops.group_top_experts(s, top_k, groups, top_groups, scoring, None if bias is None else bias.to(DEV), 1, normalize, scale)
    n64 = scores.double().numpy()
    want, _ = F.group_choice(n64, top_k, groups, top_groups, scoring, None if bias is None else bias.double().numpy(), 1, normalize, scale)
    assert np.array_equal(chosen.cpu().numpy(), want)
    exact = _weights(n64, want, scoring, normalize, scale)
    off = np.abs(weights.detach().double().cpu().numpy() - exact)
    assert (off <= 2.0 ** -18 * exact + STEP).all(), (off / exact).max()
    if normalize:
        ds, = torch.autograd.grad(weights, s, grad.to(DEV))
        g = grad.double().numpy()
        want_ds, size = np.zeros(n64.shape), np.zeros(n64.shape)
        u = g * exact
        own = u - exact / scale * u.sum(1, keepdims=True)
        np.put_along_axis(want_ds, want, own * (1 / (1 + np.exp(np.take_along_axis(n64, want, 1))) if scoring == "sigmoid" else 1.0), 1)
        np.put_along_axis(size, want, np.abs(u) + exact / scale * np.abs(u).sum(1, keepdims=True), 1)
        assert (np.abs(ds.double().cpu().numpy() - want_ds) <= 2.0 ** -17 * size + 2.0 ** -24 * np.abs(want_ds) + 2.0 ** -126).all()


@pytest.mark.parametrize("tokens", [9, 2100])
@pytest.mark.parametrize("level", [-80, -95, -110, -300, -700])
@pytest.mark.parametrize("bias", [False, True])
def test_normalised_sigmoids_that_fp32_loses(tokens, level, bias):
    """(with a bias the choice is the bias', since p is nothing beside it)"""
    g = torch.Generator().manual_seed(-level)
    scores = torch.randn(tokens, 64, generator=g) * 2 + level
    b = torch.randn(64, generator=g) if bias else None
    _check(scores, b, "sigmoid", True, 2.5)
    _check(scores, b, "sigmoid", True, 1.0, 8, 3)


@pytest.mark.parametrize("tokens", [9, 2100])
def test_normalised_sigmoids_far_apart(tokens):
    """Some of the chosen in the range of fp32 and some below it, also as weights."""
    g = torch.Generator().manual_seed(5)
    scores = torch.randn(tokens, 16, generator=g) * 60 - 60
    _check(scores, None, "sigmoid", True, 1.0, top_k=16)
    _check(scores, None, "softmax", True, 1.0, top_k=16)
    _check(scores - 300, None, "sigmoid", True, 16.0, top_k=16)


@pytest.mark.parametrize("tokens", [9, 2100])
@pytest.mark.parametrize("level", [-80, -95, -110, -300, -700])
def test_normalised_softmaxes_that_fp32_loses(tokens, level):
    """A bias that chooses none of the experts that have all of the softmax."""
    g = torch.Generator().manual_seed(-level)
    scores = torch.randn(tokens, 64, generator=g) * 2 + level
    scores[:, ::16] -= level
    b = torch.randn(64, generator=g)
    b[::16] = -100.0
    _check(scores, b, "softmax", True, 2.5)
    _check(scores, b, "softmax", True, 1.0, 8, 3)


@pytest.mark.parametrize("tokens", [9, 2100])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("scale", [1.0, 16.0, 2.0 ** 60, -2.0 ** 100])
def test_small_weights(tokens, scoring, scale):
    """p below the normal numbers of fp32, times a scale that may bring it back."""
    g = torch.Generator().manual_seed(3)
    scores = torch.randn(tokens, 32, generator=g) * 4 - 95
    b = torch.randn(32, generator=g)
    if scoring == "softmax":
        scores[:, 7] += 95
        b[7] = -100.0
    s = scores.double().numpy()
    chosen, weights = stk.ops.group_top_experts(scores.to(DEV), 8, scoring=scoring, bias=b.to(DEV), normalize=False, scale=scale)
    want, _ = F.group_choice(s, 8, 1, 1, scoring, b.double().numpy(), 1, False, scale)
    exact = _weights(s, want, scoring, False, scale)
    assert np.array_equal(chosen.cpu().numpy(), want) and (np.abs(weights.double().cpu().numpy() - exact) <= 2.0 ** -18 * np.abs(exact) + STEP).all()


@pytest.mark.parametrize("tokens", [9, 2100])
def test_rows_below_64_bits_have_no_weights(tokens):
    """Sigmoids that 64 bits do not tell from 0, a mask of the type's lowest value among them: weights of 0, and no gradient."""
    s = torch.full((tokens, 32), torch.finfo(torch.float32).min, device=DEV)
    s[1] = -800.0
    s[2] = -float("inf")
    s.requires_grad_()
    _, weights = stk.ops.group_top_experts(s, 4, 4, 2, "sigmoid")
    assert not weights.any() and not torch.autograd.grad(weights, s, torch.ones_like(weights))[0].any()
