"""Definitions, in numpy and 64 bits, of the operators around the products of a routed layer: layer norm, the router's choice
and products with 4-bit weights, with their gradients.  The library's header (include/stk_amd.h) states the same; the
reference has none of them."""
import numpy as np


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, z, 1 / deviation) of rows x [rows, size]."""
    x = np.asarray(x, dtype=np.float64)
    d = x - x.mean(axis=1, keepdims=True)
    r = 1.0 / np.sqrt((d * d).mean(axis=1, keepdims=True) + eps)
    y = z = d * r
    if weight is not None:
        y = y * np.asarray(weight, dtype=np.float64)
    if bias is not None:
        y = y + np.asarray(bias, dtype=np.float64)
    return y, z, r


def layer_norm_gradients(grad, x, weight=None, eps=1e-5):
    """(dx, dweight, dbias)."""
    grad = np.asarray(grad, dtype=np.float64)
    _, z, r = layer_norm(x, eps=eps)
    g = grad if weight is None else grad * np.asarray(weight, dtype=np.float64)
    dx = r * (g - g.mean(axis=1, keepdims=True) - z * (g * z).mean(axis=1, keepdims=True))
    return dx, (grad * z).sum(axis=0), grad.sum(axis=0)


def top_experts(scores, top_k, normalize=False):
    """(chosen, weights)."""
    s = np.asarray(scores, dtype=np.float64)
    # ties to the lower expert, NaN above every number
    ranked = np.where(np.isnan(s), np.inf, s)
    chosen = np.stack([np.lexsort((np.arange(s.shape[1]), -r, ~n)) for r, n in zip(ranked, np.isnan(s))])[:, :top_k] if len(s) else np.zeros((0, top_k), int)
    picked = np.take_along_axis(s, chosen, axis=1)
    over = picked if normalize else s
    weights = np.zeros(picked.shape)
    for t in range(len(s)):
        if np.isnan(s[t]).any() or np.isposinf(s[t]).any():
            weights[t] = np.nan
        elif not np.isneginf(s[t]).all():
            top = s[t].max()
            weights[t] = np.exp(picked[t] - top) / np.exp(over[t] - top).sum()
    return chosen.astype(np.int32), weights


def top_experts_gradient(scores, top_k, grad, normalize=False):
    """Gradient of sum(grad * weights) with respect to the scores (rows without NaN and +infinity)."""
    s, grad = np.asarray(scores, dtype=np.float64), np.asarray(grad, dtype=np.float64)
    chosen, weights = top_experts(s, top_k, normalize)
    out = np.zeros(s.shape)
    for t in range(len(s)):
        if np.isneginf(s[t]).all():
            continue
        q = np.zeros(s.shape[1])
        if normalize:
            q[chosen[t]] = weights[t]
        else:
            e = np.exp(s[t] - s[t].max())
            q = e / e.sum()
        out[t, chosen[t]] = grad[t] * weights[t]
        out[t] -= q * (grad[t] * weights[t]).sum()
    return out


def weights4(codes, scales, group, offsets=None):
    """Weights [..., inputs, outputs] of codes [..., inputs, outputs] and scales (offsets) [..., groups, outputs]."""
    rows = np.arange(codes.shape[-2]) // group
    s = np.asarray(scales, dtype=np.float64)[..., rows, :]
    c = codes.astype(np.float64)
    return s * (c - 8) if offsets is None else s * c + np.asarray(offsets, dtype=np.float64)[..., rows, :]


def gather_matmul(x, indices, bins, top_k, w):
    """Row p: x[indices[p] // top_k] @ w[e], e the first expert with bins[e] > p."""
    experts = np.searchsorted(bins, np.arange(len(indices)), side="right")
    return np.stack([x[s // top_k] @ w[e] for s, e in zip(indices, experts)]) if len(indices) else np.zeros((0, w.shape[2]))


def matmul_scatter(x, indices, bins, top_k, w, weights=None):
    """Row t: sum over its slots s = indices[p] of weights[s] * (x[p] @ w[e])."""
    out = np.zeros((len(indices) // top_k, w.shape[2]))
    experts = np.searchsorted(bins, np.arange(len(indices)), side="right")
    for p, (s, e) in enumerate(zip(indices, experts)):
        out[s // top_k] += (x[p] @ w[e]) * (1.0 if weights is None else weights[s])
    return out
