"""The example that runs layer norm, the router's choice and the 4-bit products as a layer does: examples/routed_block.py."""
import importlib.util
import os

import pytest
import torch

import stk_amd as stk

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "routed_block.py")
    spec = importlib.util.spec_from_file_location("routed_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,top_k", [(200, 2), (333, 1)])
def test_training_reaches_every_parameter(tokens, top_k, dtype):
    torch.manual_seed(1)
    m = _example()
    block = m.RoutedBlock(128, 256, 4, top_k, dtype)
    x = torch.randn(tokens, 128, device="cuda", dtype=dtype)
    block(x).float().square().mean().backward()
    for name, parameter in block.named_parameters():
        grad = parameter.grad
        assert grad.shape == parameter.shape and grad.dtype == dtype and bool(torch.isfinite(grad).all()), name
        # one chosen expert has the weight 1 whatever the scores are
        assert bool(grad.abs().sum() > 0) != (name == "router" and top_k == 1), name


def test_training_lowers_the_loss():
    torch.manual_seed(2)
    m = _example()
    block = m.RoutedBlock(128, 256, 4, 2)
    x = torch.randn(512, 128, device="cuda", dtype=torch.bfloat16)
    losses = m.train(block, x, torch.randn(512, 128, device="cuda"), 12)
    assert losses[-1] < losses[0]


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_served_block(tokens):
    """Against 64 bits with the weights that the codes stand for.  z, the choice and its weights are the block's own (each has tests of its
    own).  h is rounded to half a unit in the last place (2^-9 of it; twice that is allowed, for the fp32 sums before it), which moves the
    result by 2^-8 sum |h| |w2| at most; the sum over the choices is rounded once, and once more with x."""
    torch.manual_seed(3)
    m = _example()
    block = m.RoutedBlock(256, 384, 8, 2)
    served = m.ServedBlock(block, 64)
    x = torch.randn(tokens, 256, device="cuda", dtype=torch.bfloat16)
    got = served(x)
    with torch.no_grad():
        z, chosen, weights = (t.cpu() for t in block.choose(x))
    w1, w2 = (stk.ops.dequantize_4bit(w).double().cpu() for w in (served.w1, served.w2))
    # (the products take a group's scale times the whole codes: dequantized weights are rounded to 16 bits, half a unit each)
    near1, near2 = w1.abs() * 2.0 ** -9, w2.abs() * 2.0 ** -9
    for t in range(tokens):
        y, slack = torch.zeros(256, dtype=torch.float64), torch.zeros(256, dtype=torch.float64)
        for e, by in zip(chosen[t].tolist(), weights[t].double().tolist()):
            row = z[t].double()
            h = torch.nn.functional.gelu(row @ w1[e], approximate="tanh")
            off = 1.2 * (row.abs() @ near1[e]) + h.abs() * 2.0 ** -8
            y += by * (h @ w2[e])
            slack += by * (off @ w2[e].abs() + (h.abs() + off) @ near2[e])
        want = x[t].double().cpu() + y
        slack = slack + (y.abs() + slack) * 2.0 ** -9
        slack = slack + (want.abs() + slack) * 2.0 ** -9 + 1e-6
        assert bool(((got[t].double().cpu() - want).abs() <= slack).all()), t


def test_served_block_in_a_graph():
    torch.manual_seed(4)
    m = _example()
    served = m.ServedBlock(m.RoutedBlock(256, 256, 8, 2))
    x = torch.randn(9, 256, device="cuda", dtype=torch.bfloat16)
    graph, out = m.captured(served, x)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, served(x))
