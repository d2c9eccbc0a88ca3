"""Products with weights of 4 bits and a scale for every group of inputs: the serving form of the experts' products.

A decoding step reads the weights of every expert that is hit for a handful of rows, so that what it takes is the bytes of
those weights; here they are a quarter of the 16-bit ones and become 16-bit values in registers.  The products take the routing of
stk.ops.route as it is and pad nothing.  The reference has no counterpart; in a layer they stand where
stk.ops.gather_sdd and stk.ops.dsd_scatter are with 16-bit weights."""
from collections import namedtuple

import torch

from stk_amd.backend import autocast, hip_kernels
from stk_amd.backend.autograd import applies

# packed, scales, offsets (or None): device tensors in the layout of the products, [experts, ...]; experts: None for a single matrix
Weights4 = namedtuple("Weights4", "packed scales offsets experts inputs outputs group_size")


def _batched(t, dims):
    return t if t is None or t.dim() == dims else t.unsqueeze(0)


def _no_gradient(*tensors):
    if applies(*tensors):
        raise NotImplementedError("stk_amd: 4-bit weights are for inference: their products have no gradient and are not traced or transformed")


def _operand(x):
    """x as the products of this package see it: under autocast in its type."""
    return x.to(torch.get_autocast_gpu_dtype()) if autocast.casts(x) else x


@torch.no_grad()
def pack_4bit(codes, scales, group_size, offsets=None):
    """Weights4 of given codes 0 .. 15 (uint8, one a byte) [inputs, outputs] or [experts, inputs, outputs] on the GPU: weight = scale * (code - 8), or
    scale * code + offset where offsets are given.  scales and offsets are float16 or bfloat16 [(experts,) groups, outputs], groups =
    ceil(inputs / group_size); group_size 32, 64 or a multiple of 128."""
    assert codes.dim() in (2, 3) and scales.dim() == codes.dim()
    packed = hip_kernels.pack_4bit(_batched(codes, 3), _batched(scales, 3), group_size, _batched(offsets, 3))
    return Weights4(*packed, codes.size(0) if codes.dim() == 3 else None, codes.size(-2), codes.size(-1), group_size)


@torch.no_grad()
def quantize_4bit(weights, group_size=128, offsets=False, dtype=None):
    """Weights4 nearest to weights [inputs, outputs] or [experts, inputs, outputs] (any strides: the experts' slices of
    [inputs, experts * outputs] are weights.view(inputs, experts, outputs).transpose(0, 1)).

    offsets=False: scale = max |w| of a group / 7.  offsets=True: scale = (max - min) / 15 and the smallest weight as the offset.  A group
    with a NaN or an infinity, or with weights too large for the scales' type, becomes NaN as a whole.  dtype:
    float16 or bfloat16, the type of the scales and of the rows that are multiplied; default: that of the weights."""
    assert weights.dim() in (2, 3)
    codes, scales, from_ = hip_kernels.quantize_4bit(_batched(weights, 3), group_size, offsets, dtype or weights.dtype)
    packed = hip_kernels.pack_4bit(codes, scales, group_size, from_)
    return Weights4(*packed, weights.size(0) if weights.dim() == 3 else None, weights.size(-2), weights.size(-1), group_size)


def dequantize_4bit(w):
    """The weights [inputs, outputs] or [experts, inputs, outputs] that w stands for, in the type of its scales."""
    out = hip_kernels.dequantize_4bit(w.packed, w.scales, w.offsets, w.inputs, w.outputs, w.group_size)
    return out[0] if w.experts is None else out


def matmul_4bit(x, w, activation=None):
    """activation(x @ w) for x [..., inputs] of w's type and a single matrix w; the activations are those of stk.ops.sdd_fused, applied to the
    fp32 sums.  A row with an infinity or a NaN gives NaN throughout, here and in the products below.  Under autocast x is cast to its type
    like the operands of the other products.  Inference only: raises where x needs a gradient."""
    assert isinstance(w, Weights4) and w.experts is None
    _no_gradient(x)
    x = _operand(x)
    rows = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    out = hip_kernels.matmul_4bit(rows, w.packed, w.scales, w.offsets, w.inputs, w.outputs, w.group_size, activation)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], w.outputs)


def gather_matmul_4bit(x, route, w, activation=None):
    """activation(x[token] @ w[expert]) for every slot of the routing: x [tokens, inputs] -> [slots, outputs], rows in the order of
    route.indices (by expert, without padding, whatever blocking the routing was made with).  Inference only."""
    assert isinstance(w, Weights4) and w.experts is not None
    _no_gradient(x)
    return hip_kernels.gather_matmul_4bit(_operand(x), route.indices, route.bins, route.top_k, w.packed, w.scales, w.offsets, w.inputs, w.outputs, w.group_size,
                                          activation)


def matmul_4bit_scatter(x, route, w, weights=None):
    """The way back: x [slots, inputs], rows in the order of route.indices -> [tokens, outputs], each token's top_k products
    x @ w[expert], multiplied by weights [tokens, top_k] (fp32, or None), added up in fp32 in the order of the choices and rounded
    once.  Inference only."""
    assert isinstance(w, Weights4) and w.experts is not None
    _no_gradient(x, weights)
    return hip_kernels.matmul_4bit_scatter(_operand(x), route.indices, route.bins, route.top_k, w.packed, w.scales, w.offsets, w.inputs, w.outputs, w.group_size,
                                           weights)
