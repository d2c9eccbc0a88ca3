"""A pre-norm block with a dropless mixture of experts: trained with the block-sparse products, then served from 4-bit weights.

    python examples/routed_block.py [--tokens 8192] [--hidden 1024] [--ffn 4096] [--experts 64] [--top-k 2] [--steps 20]

x + sum over the chosen experts of weight * (gelu(norm(x) w1[expert]) w2[expert]).  Random weights, random data."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import stk_amd as stk

BLOCK = 128


class RoutedBlock(torch.nn.Module):
    def __init__(self, hidden, ffn, experts, top_k, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.ffn, self.experts, self.top_k = ffn, experts, top_k
        new = dict(dtype=dtype, device=device)
        self.norm_weight, self.norm_bias = torch.nn.Parameter(torch.ones(hidden, **new)), torch.nn.Parameter(torch.zeros(hidden, **new))
        self.router = torch.nn.Parameter(torch.randn(hidden, experts, **new) * hidden ** -0.5)
        self.w1 = torch.nn.Parameter(torch.randn(hidden, experts * ffn, **new) * hidden ** -0.5)
        self.w2 = torch.nn.Parameter(torch.randn(experts * ffn, hidden, **new) * ffn ** -0.5)

    def choose(self, x):
        """(normalised rows, chosen experts, their weights)"""
        z = stk.ops.layer_norm(x, self.norm_weight, self.norm_bias)
        return z, *stk.ops.top_experts(z @ self.router, self.top_k, normalize=True)

    def forward(self, x):
        z, chosen, weights = self.choose(x)
        r = stk.ops.route(chosen, self.experts, BLOCK)
        padded = stk.ops.padded_gather(z, r)
        topo = stk.ops.dmoe_topology(r.padded_bins, BLOCK, padded.size(0) // BLOCK, self.ffn // BLOCK, dtype=x.dtype)
        h = stk.ops.sdd_fused(padded, self.w1, topo, "gelu_tanh", save_sums=True)
        return x + stk.ops.padded_scatter(stk.ops.dsd(h, self.w2), r, weights)


class ServedBlock:
    """The same block with its experts' weights in 4 bits.  Nothing in a call waits for the device, so that it can be captured into a
    HIP graph."""

    @torch.no_grad()
    def __init__(self, block, group_size=128):
        self.block = block
        hidden = block.w1.size(0)
        self.w1 = stk.ops.quantize_4bit(block.w1.view(hidden, block.experts, block.ffn).transpose(0, 1), group_size)
        self.w2 = stk.ops.quantize_4bit(block.w2.view(block.experts, block.ffn, hidden), group_size)

    @torch.no_grad()
    def __call__(self, x):
        z, chosen, weights = self.block.choose(x)
        r = stk.ops.route(chosen, self.block.experts, 1, padded_rows=chosen.numel())   # (the products pad nothing)
        h = stk.ops.gather_matmul_4bit(z, r, self.w1, "gelu_tanh")
        return x + stk.ops.matmul_4bit_scatter(h, r, self.w2, weights)


def train(block, x, target, steps, lr=1e-3):
    """Losses of `steps` steps on one batch."""
    optimizer = torch.optim.Adam(block.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = torch.nn.functional.mse_loss(block(x).float(), target)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def captured(served, x):
    """(graph, result) of served(x)"""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        served(x)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = served(x)
    return graph, out


def microseconds(call, times=20):
    call()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(times):
        call()
    end.record()
    end.synchronize()
    return start.elapsed_time(end) * 1000 / times


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 8192), ("hidden", 1024), ("ffn", 4096), ("experts", 64), ("top-k", 2), ("steps", 20)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args()
    torch.manual_seed(0)
    block = RoutedBlock(a.hidden, a.ffn, a.experts, a.top_k)
    x = torch.randn(a.tokens, a.hidden, device="cuda", dtype=torch.bfloat16)
    losses = train(block, x, torch.randn(a.tokens, a.hidden, device="cuda"), a.steps)
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")

    served = ServedBlock(block)
    with torch.no_grad():
        want = block(x).float()
        off = (served(x).float() - want).norm() / (want - x.float()).norm()
    print(f"4-bit weights: the experts' part differs by {off:.3f} of its norm")
    for tokens in (1, 16, 128):
        few = x[:tokens].clone()
        graph, _ = captured(served, few)
        with torch.no_grad():
            print(f"{tokens:4d} tokens: {microseconds(graph.replay):7.1f} us from 4-bit weights (a graph), {microseconds(lambda: block(few)):7.1f} us from 16-bit ones")


if __name__ == "__main__":
    main()
