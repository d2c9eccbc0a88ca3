"""More tokens than one launch of the router among groups takes: in parts, of which each token's results are those of a call of its own."""
import pytest
import torch

import stk_amd as stk

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("groups", [17, 1])
def test_many_tokens(groups):
    """2^26 tokens and some: with a wavefront each more threads than a launch may have."""
    tokens, experts = 2 ** 26 + 5, 17
    scores = torch.empty(tokens, experts, dtype=torch.bfloat16, device=DEV)
    for r in range(0, tokens, 1 << 24):
        part = scores[r:r + (1 << 24)]
        part.copy_(torch.randn(part.shape, dtype=torch.bfloat16, device=DEV, generator=torch.Generator(device=DEV).manual_seed(r)))
    scores.requires_grad_()
    grad = torch.ones(1, 1, device=DEV).expand(tokens, 1)
    chosen, weights = stk.ops.group_top_experts(scores, 1, groups, 1, "sigmoid", None, 1, False, 1.0)
    ds, = torch.autograd.grad(weights, scores, grad)
    assert torch.equal(scores.detach().gather(1, chosen.long())[:, 0], scores.detach().amax(1))
    for at in [slice(0, 3000), slice(tokens - 3000, tokens)] + [slice(k * (1 << 24) - 1500, k * (1 << 24) + 1500) for k in (1, 2, 3)]:
        part = scores.detach()[at].clone().requires_grad_()
        c, w = stk.ops.group_top_experts(part, 1, groups, 1, "sigmoid", None, 1, False, 1.0)
        d, = torch.autograd.grad(w, part, torch.ones_like(w))
        assert torch.equal(chosen[at], c) and torch.equal(weights[at], w) and torch.equal(ds[at], d), at
