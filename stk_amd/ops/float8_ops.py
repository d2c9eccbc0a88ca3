"""Products in 8-bit floating point (e4m3) with a scale for every block of 128: half the bytes of 16-bit operands, and twice the rate of the matrix units.

Stored weights have a scale for every 128 inputs x 128 outputs; the rows they are multiplied with are quantised within the call, every 128 values
of a row with a scale of their own, the smallest power of two 2^e (e >= -126) with max |x| <= 448 2^e.  Sums are fp32.  The reference has no counterpart;
in a layer the products of stored weights stand where stk.ops.gather_sdd and stk.ops.dsd_scatter are with 16-bit weights, and linear_8bit where
stk.ops.sdd and stk.ops.dsd are on the padded layout of a routing."""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from stk_amd.backend import autocast, hip_kernels
from stk_amd.backend.autograd import applies, seen_by_python_only

# packed, scales: device tensors in the layout of the products, [experts, ...]; experts: None for a single matrix
Weights8 = namedtuple("Weights8", "packed scales experts inputs outputs")


def _batched(t):
    return t if t.dim() == 3 else t.unsqueeze(0)


def _no_gradient(*tensors):
    if applies(*tensors):
        raise NotImplementedError("stk_amd: stored 8-bit weights are for inference: their products have no gradient and are not traced or transformed; "
                                  "linear_8bit has one")


def _operand(x):
    """x as the products of this package see it: under autocast in its type."""
    return x.to(torch.get_autocast_gpu_dtype()) if autocast.casts(x) else x


@torch.no_grad()
def pack_8bit(codes, scales):
    """Weights8 of given codes (float8_e4m3fn) [inputs, outputs] or [experts, inputs, outputs] on the GPU: weight = scale * code.  scales
    [(experts,) ceil(inputs / 128), ceil(outputs / 128)], float32 of any value or float8_e8m0fnu (powers of two, which the matrix units apply)."""
    assert codes.dim() in (2, 3) and scales.dim() == codes.dim()
    packed = hip_kernels.pack_8bit(_batched(codes), _batched(scales))
    return Weights8(*packed, codes.size(0) if codes.dim() == 3 else None, codes.size(-2), codes.size(-1))


@torch.no_grad()
def quantize_8bit(weights):
    """Weights8 nearest to weights [inputs, outputs] or [experts, inputs, outputs] (float16, bfloat16 or float32, any strides: the experts' slices of
    [inputs, experts * outputs] are weights.view(inputs, experts, outputs).transpose(0, 1)), with scales that are powers of two.  A block with a
    NaN or an infinity becomes NaN as a whole."""
    assert weights.dim() in (2, 3)
    packed = hip_kernels.quantize_8bit(_batched(weights))
    return Weights8(*packed, weights.size(0) if weights.dim() == 3 else None, weights.size(-2), weights.size(-1))


def dequantize_8bit(w, dtype=torch.bfloat16):
    """The weights [inputs, outputs] or [experts, inputs, outputs] that w stands for, each rounded once to dtype."""
    out = hip_kernels.dequantize_8bit(w.packed, w.scales, w.inputs, w.outputs, dtype)
    return out[0] if w.experts is None else out


def matmul_8bit(x, w, activation=None):
    """activation(x @ w) for x [..., inputs], float16 or bfloat16, and a single matrix w; the activations are those of stk.ops.sdd_fused, applied to the
    fp32 sums; the result is of x's type.  A row with an infinity or a NaN gives NaN throughout, here and in the products below.  Under autocast x is cast to its
    type like the operands of the other products.  Inference only: raises where x needs a gradient."""
    assert isinstance(w, Weights8) and w.experts is None
    _no_gradient(x)
    x = _operand(x)
    rows = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    out = hip_kernels.matmul_8bit(rows, w.packed, w.scales, w.inputs, w.outputs, activation)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], w.outputs)


def gather_matmul_8bit(x, route, w, activation=None):
    """activation(x[token] @ w[expert]) for every slot of the routing: x [tokens, inputs] -> [slots, outputs], rows in the order of
    route.indices (by expert, without padding, whatever blocking the routing was made with).  Inference only."""
    assert isinstance(w, Weights8) and w.experts is not None
    _no_gradient(x)
    return hip_kernels.gather_matmul_8bit(_operand(x), route.indices, route.bins, route.top_k, w.packed, w.scales, w.inputs, w.outputs, activation)


def matmul_8bit_scatter(x, route, w, weights=None):
    """The way back: x [slots, inputs], rows in the order of route.indices -> [tokens, outputs], each token's top_k products
    x @ w[expert], multiplied by weights [tokens, top_k] (fp32, or None), added up in fp32 in the order of the choices and rounded
    once.  Inference only."""
    assert isinstance(w, Weights8) and w.experts is not None
    _no_gradient(x, weights)
    return hip_kernels.matmul_8bit_scatter(_operand(x), route.indices, route.bins, route.top_k, w.packed, w.scales, w.inputs, w.outputs, weights)


class _Linear8(torch.autograd.Function):
    """What forward-mode differentiation and transforms refuse and torch.jit.trace records; otherwise the native function runs."""

    @staticmethod
    def forward(ctx, x, w, bins):
        out, saved = hip_kernels.linear_8bit_forward(x, w, bins, *ctx.needs_input_grad[:2])
        ctx.save_for_backward(*saved, bins)
        ctx.shapes = x.shape, w.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        *saved, bins = ctx.saved_tensors
        return *hip_kernels.linear_8bit_backward(grad, saved, bins, *ctx.shapes, *ctx.needs_input_grad[:2]), None


def linear_8bit(x, w, route=None):
    """x @ w with both operands quantised within the call, and gradients computed the same way: the product of a training step.

    x [..., inputs] and w [inputs, outputs]; or, with a routing, the rows of its padded layout (stk.ops.padded_gather; a blocking of 128 or a
    multiple) and w [experts, inputs, outputs]: every row times its expert's matrix, zeros in rows behind the last expert's.  x and w both float16 or both
    bfloat16 (w of any strides), the result of their type; under autocast both are cast to its type.
    w is quantised with a scale for every 128 x 128 values, x for every 128 of a row.  The gradient of x is grad @ w^T with the same 8-bit weights and grad quantised
    for every 128 of a row; that of w is x^T @ grad with both quantised for every 128 rows of a column.  Scales are powers of two.  What is kept
    for the backward pass is 8-bit: the columns of x and the transpose of w.  A block with an infinity or a NaN is NaN as a whole."""
    bins = None
    if route is not None:
        assert route.blocking % 128 == 0, "linear_8bit: a routing with a blocking of 128 or a multiple"
        assert x.dim() == 2 and x.size(0) == route.row_slots.numel(), "linear_8bit: the rows of the routing's padded layout"
        bins = route.padded_bins
    x, w = _operand(x), _operand(w)
    if seen_by_python_only():
        return _Linear8.apply(x, w, bins)
    return hip_kernels.linear_8bit(x, w, bins)
