"""Which experts a router chooses among groups where fp32 keys, margins or sums reach the ends of their range: the definition's, whatever they are."""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _same(scores, bias, top_k, groups, top_groups, best, scoring):
    got, _ = stk.ops.group_top_experts(scores.to(DEV), top_k, groups, top_groups, scoring, None if bias is None else bias.to(DEV), best)
    n64 = scores.double().numpy()
    if bias is None and best == 1:   # (p has the order of the scores; in 64 bits those of scores next to 0 are equal: choose by c of the scores' own size)
        n64 = n64 / np.abs(n64).max()
    want, _ = F.group_choice(n64, top_k, groups, top_groups, scoring, None if bias is None else bias.double().numpy(), best)
    wrong = np.argwhere(got.cpu().numpy() != want)
    assert not wrong.size, (wrong[0].tolist(), len(wrong))


@pytest.mark.parametrize("tokens", [60, 2100])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("unit", [2.0 ** -149, 2.0 ** -140, 2.0 ** -130, 2.0 ** -126])
def test_subnormal_scores(tokens, scoring, unit):
    """Scores of a few units of the smallest steps of fp32, of both signs, which only their order tells apart."""
    g = torch.Generator().manual_seed(7)
    scores = (torch.randint(-40, 41, (tokens, 64), generator=g).double() * unit).float()
    scores[0, :], scores[0, 5], scores[0, 9] = 0.0, 3 * unit, 9 * unit
    scores[1] = torch.arange(64).double() * -unit
    for groups, top_groups, best in ((1, 1, 1), (8, 3, 1), (8, 3, 2)):
        _same(scores, None, 8, groups, top_groups, best, scoring)
        _same(scores, None, 1, groups, top_groups, best, scoring)


@pytest.mark.parametrize("tokens", [200, 2100])
@pytest.mark.parametrize("bias", [False, True])
def test_sums_of_sigmoids_below_the_normal_numbers(tokens, bias):
    """A group's two best around 2^-126, where one of them may have no normal number and the other one."""
    g = torch.Generator().manual_seed(3)
    scores = torch.randn(tokens, 64, generator=g) * 0.7 - 87.3
    b = torch.randn(64, generator=g) * 2.0 ** -127 if bias else None
    _same(scores, b, 8, 8, 3, 2, "sigmoid")
    _same(scores, b, 8, 8, 3, 1, "sigmoid")


@pytest.mark.parametrize("tokens", [60, 2100])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_biases_whose_sum_leaves_fp32(tokens, scoring):
    """Groups whose two best add up to more than fp32 has, above and below."""
    scores = torch.randn(tokens, 16, generator=torch.Generator().manual_seed(4))
    bias = torch.tensor([3.2, 3.0, -1.0, -2.0, 3.3, 3.1, -1.1, -2.2, 2.0, 1.0, 0.5, -2.5, 1.5, 0.7, 0.2, -2.6]) * 1e38
    _same(scores, bias, 2, 4, 1, 2, scoring)
    below = torch.tensor([-3.0, -3.3, -3.31, -3.32, 0.0, 1.0, 2.0, 3.0, -2.9, -3.1, -3.2, -3.25, -2.7, -2.8, -3.3, -3.32]) * 1e38
    _same(scores, below, 1, 4, 3, 2, scoring)
    _same(scores, below, 12, 4, 3, 2, scoring)
