"""GPU parity of the 8-bit product of a training step and its gradients against the 64-bit definition.

Whole numbers of at most 8 are exact through quantisation (of rows, columns and blocks alike), products and sums (test_gpu_float8.py), so that results
are the roundings of exact ones: equal bits, and differences of the product give its gradients.  Other values: oracle.float8_oracle.slack_of and half
a unit in the last place.
"""
import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F
from tests.test_gpu_float8 import DEV, _check, _n64, _whole

pytestmark = pytest.mark.gpu
SIZES = [(1, 128, 128), (128, 128, 128), (5, 1, 1), (130, 70, 200), (300, 1151, 96), (64, 256, 513), (1000, 640, 1030), (2100, 2048, 2304), (129, 4096, 257), (257, 65, 4096)]


def _step(x, w, grad, route=None):
    x, w = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = stk.ops.linear_8bit(x, w, route)
    return (y.detach(), *torch.autograd.grad(y, (x, w), grad.to(DEV)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_whole_numbers(rows, inputs, outputs, dtype):
    g = torch.Generator().manual_seed(rows + inputs)
    x, w, grad = _whole((rows, inputs), g, 4), _whole((inputs, outputs), g, 4), _whole((rows, outputs), g, 2)
    y, dx, dw = _step(x.to(dtype), w.to(dtype), grad.to(dtype))
    for got, want in ((y, x.double() @ w.double()), (dx, grad.double() @ w.double().t()), (dw, x.double().t() @ grad.double())):
        assert torch.equal(got.cpu(), want.float().to(dtype))
    # what is not wanted changes nothing
    only_x, only_w = x.to(dtype).to(DEV).requires_grad_(), w.to(dtype).to(DEV).requires_grad_()
    assert torch.equal(torch.autograd.grad(stk.ops.linear_8bit(only_x, only_w.detach()), only_x, grad.to(dtype).to(DEV))[0], dx)
    assert torch.equal(torch.autograd.grad(stk.ops.linear_8bit(only_x.detach(), only_w), only_w, grad.to(dtype).to(DEV))[0], dw)
    with torch.no_grad():
        assert torch.equal(stk.ops.linear_8bit(only_x, only_w), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,inputs,outputs", [(100, 300, 200), (300, 130, 400)])
def test_against_the_definition(rows, inputs, outputs, dtype):
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, inputs, generator=g) * torch.exp(torch.randn(inputs, generator=g))).to(dtype)
    w, grad = (torch.randn(inputs, outputs, generator=g) * inputs ** -0.5).to(dtype), (torch.randn(rows, outputs, generator=g) * 0.01).to(dtype)
    y, dx, dw = _step(x, w, grad)
    wq = F.quantised(_n64(w), 128, 128)[0]
    for got, a, b in ((y, F.quantised(_n64(x), 1, 128)[0], wq), (dx, F.quantised(_n64(grad), 1, 128)[0], wq.T),
                      (dw, F.quantised(_n64(x), 128, 1)[0].T, F.quantised(_n64(grad), 128, 1)[0])):
        _check(got, a @ b, F.slack_of(a, b), dtype)


def test_differences():
    """<y(x + a, w + b) - y(x, w), g> is <dx, a> + <dw, b> + <a b, g>, exactly in whole numbers whose 16-bit results are exact."""
    g = torch.Generator().manual_seed(0)
    x, w, grad = _whole((40, 32), g, 2), _whole((32, 24), g, 2), _whole((40, 24), g, 1)
    a, b = _whole((40, 32), g, 1), _whole((32, 24), g, 1)
    y, dx, dw = (t.double().cpu() for t in _step(x.half(), w.half(), grad.half()))
    moved = stk.ops.linear_8bit((x + a).half().to(DEV), (w + b).half().to(DEV)).double().cpu()
    assert ((moved - y) * grad).sum() == (dx * a).sum() + (dw * b).sum() + ((a.double() @ b.double()) * grad).sum()


ROUTED = [(200, 4, 2, 128, 256, "any", 0), (1000, 8, 1, 300, 200, "half", 1), (5, 16, 2, 96, 130, "any", 0), (700, 3, 1, 640, 1000, "one", 300), (3000, 5, 2, 256, 1024, "any", 1000),
          (1, 2, 1, 64, 64, "any", 0), (40, 200, 2, 128, 64, "any", 128)]


@pytest.mark.parametrize("blocking", [128, 256])
@pytest.mark.parametrize("tokens,experts,top_k,inputs,outputs,how,behind", ROUTED)
def test_experts(tokens, experts, top_k, inputs, outputs, how, behind, blocking):
    """The rows of a routing's padded layout, also with more rows than it needs, whose contents have no say but in the gradients' blocks of 128."""
    g = torch.Generator().manual_seed(tokens)
    dtype = torch.bfloat16
    high = {"any": experts, "half": max(1, experts // 2), "one": 1}[how]
    top = torch.randint(0, high, (tokens, top_k), generator=g, dtype=torch.int32).to(DEV)
    need = int(stk.ops.route(top, experts, blocking).padded_bins[-1])
    r = stk.ops.route(top, experts, blocking, need + behind)
    slots = r.row_slots.cpu().long()
    x = _whole((tokens, inputs), g, 4)[slots.clamp(min=0) // top_k] * (slots >= 0).unsqueeze(1)
    rows, bins = x.size(0), [0] + r.padded_bins.cpu().tolist()
    assert rows == need + behind
    w, grad = _whole((experts, inputs, outputs), g, 4), _whole((rows, outputs), g, 2)
    x[need:] = 3
    y, dx, dw = _step(x.to(dtype), w.to(dtype), grad.to(dtype), r)
    want_y, want_dx, want_dw = torch.zeros(rows, outputs).double(), torch.zeros(rows, inputs).double(), torch.zeros(w.shape).double()
    for e in range(experts):
        at = slice(bins[e], bins[e + 1])
        want_y[at], want_dx[at], want_dw[e] = x[at].double() @ w[e].double(), grad[at].double() @ w[e].double().t(), x[at].double().t() @ grad[at].double()
    for name, got, want in (("y", y, want_y), ("dx", dx, want_dx), ("dw", dw, want_dw)):
        assert torch.equal(got.cpu(), want.float().to(dtype)), name


def test_shapes_and_strides():
    g = torch.Generator().manual_seed(2)
    x, w, grad = _whole((3, 5, 72), g, 4), _whole((72, 40), g, 4), _whole((3, 5, 40), g, 2)
    want = _step(x.view(15, 72).bfloat16(), w.bfloat16(), grad.view(15, 40).bfloat16())
    for xs, ws, gs in ((x.bfloat16(), w.bfloat16(), grad.bfloat16()), (x.transpose(0, 1).contiguous().transpose(0, 1).bfloat16(), w.t().contiguous().t().bfloat16(),
                                                                       grad.transpose(1, 2).contiguous().transpose(1, 2).bfloat16())):
        y, dx, dw = _step(xs, ws, gs)
        assert torch.equal(y.view(15, 40), want[0]) and torch.equal(dx.reshape(15, 72), want[1]) and torch.equal(dw, want[2])
    one = _step(x[0, 0].bfloat16(), w.bfloat16(), grad[0, 0].bfloat16())
    assert torch.equal(one[0], want[0][0]) and torch.equal(one[1], want[1][0])
    # a gradient that is one row for all
    y, dx, dw = _step(x.view(15, 72).bfloat16(), w.bfloat16(), grad.view(15, 40)[:1].bfloat16().expand(15, 40))
    again = _step(x.view(15, 72).bfloat16(), w.bfloat16(), grad.view(15, 40)[:1].repeat(15, 1).bfloat16())
    assert torch.equal(dx, again[1]) and torch.equal(dw, again[2])


def test_no_rows():
    y, dx, dw = _step(torch.empty(0, 64).bfloat16(), torch.ones(64, 32).bfloat16(), torch.empty(0, 32).bfloat16())
    assert y.shape == (0, 32) and dx.shape == (0, 64) and torch.equal(dw.cpu(), torch.zeros(64, 32).bfloat16())


def test_blocks_that_are_not_numbers():
    g = torch.Generator().manual_seed(5)
    x, w, grad = torch.randn(300, 300, generator=g).bfloat16(), torch.randn(300, 300, generator=g).bfloat16(), torch.randn(300, 300, generator=g).bfloat16()
    x[140, 130] = float("inf")
    y, dx, dw = (t.cpu() for t in _step(x, w, grad))
    assert y[140].isnan().all() and torch.isfinite(y[:140]).all() and torch.isfinite(y[141:]).all()
    assert torch.isfinite(dx).all() and dw[130].isnan().all() and torch.isfinite(dw[:130]).all() and torch.isfinite(dw[131:]).all()
    x[140, 130], grad[7, 299] = 0, float("nan")
    y, dx, dw = (t.cpu() for t in _step(x, w, grad))
    assert dx[7].isnan().all() and torch.isfinite(dx[:7]).all() and torch.isfinite(dx[8:]).all() and dw[:, 299].isnan().all() and torch.isfinite(dw[:, :299]).all()


def test_same_bits_every_time():
    g = torch.Generator().manual_seed(6)
    x, w, grad = torch.randn(700, 513, generator=g).bfloat16(), torch.randn(513, 900, generator=g).bfloat16(), torch.randn(700, 900, generator=g).bfloat16()
    first = _step(x, w, grad)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _step(x, w, grad)))


def test_autocast():
    g = torch.Generator().manual_seed(7)
    x, w, grad = _whole((20, 64), g, 4), _whole((64, 32), g, 4), _whole((20, 32), g, 2)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = stk.ops.linear_8bit(xs, ws)
    dx, dw = torch.autograd.grad(y, (xs, ws), grad.bfloat16().to(DEV))
    want = _step(x.bfloat16(), w.bfloat16(), grad.bfloat16())
    assert y.dtype == torch.bfloat16 and dx.dtype == dw.dtype == torch.float32
    assert torch.equal(y, want[0]) and torch.equal(dx, want[1].float()) and torch.equal(dw, want[2].float())


def test_streams_and_graphs():
    """A whole step on another stream, and captured and replayed."""
    g = torch.Generator().manual_seed(8)
    x, w, grad = (torch.randn(s, generator=g).bfloat16().to(DEV) for s in ((300, 200), (200, 400), (300, 400)))
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        y = stk.ops.linear_8bit(xs, ws)
        return (y.detach(), *torch.autograd.grad(y, (xs, ws), grad))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for replay in range(3):
        with torch.no_grad():
            xs.copy_(torch.randn(xs.shape, generator=g)), ws.copy_(torch.randn(ws.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.clone() for t in got]
        xs, ws = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        assert all(torch.equal(a, b) for a, b in zip(fresh, step())), replay


def test_refusals():
    x, w = torch.zeros(128, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(64, 32, dtype=torch.bfloat16, device=DEV)
    r = stk.ops.route(torch.zeros(100, 1, dtype=torch.int32, device=DEV), 2, 128)
    small = stk.ops.route(torch.zeros(128, 1, dtype=torch.int32, device=DEV), 2, 64)
    for call in (lambda: stk.ops.linear_8bit(x[:, :63], w), lambda: stk.ops.linear_8bit(x, w[None]), lambda: stk.ops.linear_8bit(x, w, r),
                 lambda: stk.ops.linear_8bit(x, w[None].expand(3, 64, 32), r), lambda: stk.ops.linear_8bit(x[:127], w[None].expand(2, 64, 32), r),
                 lambda: stk.ops.linear_8bit(x, w[None].expand(2, 64, 32), small)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: stk.ops.linear_8bit(x.float(), w.float()), lambda: stk.ops.linear_8bit(x, w.half()), lambda: stk.ops.linear_8bit(x.double(), w.double())):
        with pytest.raises(NotImplementedError):
            call()
    xs = x.clone().requires_grad_()
    dx, = torch.autograd.grad(stk.ops.linear_8bit(xs, w).sum(), xs, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("tokens,experts,hidden,ffn", [(300, 8, 96, 200), (6000, 16, 1032, 1544)])
def test_a_routed_layer(tokens, experts, hidden, ffn):
    """A router's choice among groups, the padded layout, both products and the way back, trained, against the same layer with every expert's products by
    themselves: blocks are the same, so that results and gradients differ by what sums in another order differ, 2^-8 of the largest."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(tokens, hidden, generator=g).bfloat16().to(DEV)
    scores, bias = torch.randn(tokens, experts, generator=g).to(DEV), (torch.randn(experts, generator=g) * 0.1).to(DEV)
    w1 = (torch.randn(experts, hidden, ffn, generator=g) * hidden ** -0.5).bfloat16().to(DEV)
    w2 = (torch.randn(experts, ffn, hidden, generator=g) * ffn ** -0.5).bfloat16().to(DEV)
    grad = torch.randn(tokens, hidden, generator=g).bfloat16().to(DEV)

    def layer(product):
        leaves = [t.detach().clone().requires_grad_() for t in (x, scores, w1, w2)]
        a, s, u, v = leaves
        chosen, weights = stk.ops.group_top_experts(s, 2, groups=4, top_groups=2, bias=bias)
        r = stk.ops.route(chosen, experts, 128)
        h = torch.relu(product(stk.ops.padded_gather(a, r), u, r))
        out = stk.ops.padded_scatter(product(h, v, r), r, weights)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))

    def apart(rows, w, r):
        ends = [0] + r.padded_bins.tolist()
        parts = [stk.ops.linear_8bit(rows[ends[e]:ends[e + 1]], w[e]) for e in range(experts)]
        return torch.cat(parts + [rows.new_zeros(rows.size(0) - ends[-1], w.size(2))])

    for got, want in zip(layer(stk.ops.linear_8bit), layer(apart)):
        assert (got.double() - want.double()).abs().max() <= 2.0 ** -8 * want.double().abs().max()
