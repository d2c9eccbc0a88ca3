"""Layer norm of token rows, the step in front of a routed layer's router and experts.  The reference has no such
operator; its callers use torch's."""
import torch
from torch.autograd.function import once_differentiable

from stk_amd.backend import hip_kernels
from stk_amd.backend.autograd import seen_by_python_only


class _LayerNorm(torch.autograd.Function):
    """What forward-mode differentiation and transforms refuse and torch.jit.trace records; otherwise the native function runs."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, statistics = hip_kernels.layer_norm(x, weight, bias, eps, with_statistics=True)
        ctx.save_for_backward(x, weight, bias, statistics)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, statistics = ctx.saved_tensors
        return (*hip_kernels.layer_norm_backward(grad, x, statistics, weight, bias, *ctx.needs_input_grad[:3]), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x [..., size] on the GPU.

    x float16, bfloat16 or float32; weight and bias [size] (or None) of x's type or float32, both of one type.  Statistics and sums
    are fp32 and every result is rounded once, to the type of what it belongs to.  The gradients of x, weight and bias
    have the same bits every time.  x may have any strides (rows that are not one distance apart, or whose values are not next to each
    other, are copied first); the result is contiguous."""
    if seen_by_python_only():
        return _LayerNorm.apply(x, weight, bias, eps)
    return hip_kernels.layer_norm_graph(x, weight, bias, eps)
