"""64-bit definitions of the 8-bit floating-point formats and products and of a router's choice among groups of experts, in numpy."""
import numpy as np

BLOCK = 128


def e4m3(v):
    """Values of at most 448 rounded to the nearest with 3 bits of mantissa down to 2^-6 and a step of 2^-9 below, ties to even."""
    _, exponent = np.frexp(v)
    step = np.ldexp(1.0, np.maximum(exponent, -5) - 4)
    return np.rint(v / step) * step


def power_of(most):
    """The smallest 2^e, e >= -126, with most <= 448 2^e."""
    mantissa, exponent = np.frexp(np.where(np.isfinite(most), most, 1.0))     # mantissa in [0.5, 1), 448 = 0.875 2^9
    e = np.where(most == 0, -126, exponent - 9 + (mantissa > 0.875))
    return np.ldexp(1.0, np.maximum(e, -126))


def quantised(x, rows, cols):
    """(values that the codes stand for, scale of every element) of x under one power of two for every rows x cols block."""
    out, scales = np.empty(x.shape), np.empty(x.shape)
    for r in range(0, x.shape[0], rows):
        for c in range(0, x.shape[1], cols):
            part = x[r:r + rows, c:c + cols]
            s = power_of(np.abs(part).max())
            out[r:r + rows, c:c + cols] = e4m3(part / s) * s if np.isfinite(part).all() else np.nan
            scales[r:r + rows, c:c + cols] = s
    return out, scales


def blocks_of(scales, inputs, outputs):
    """scales [input blocks, output blocks] for every weight."""
    return np.repeat(np.repeat(scales, BLOCK, 0), BLOCK, 1)[:inputs, :outputs]


def slack_of(a, b):
    """What the sums of a @ b may be off: in every block of 128 products each of the 127 others may lose 2^-13 of the largest; then fp32 sums of the blocks."""
    total = np.zeros((a.shape[0], b.shape[1]))
    for k in range(0, a.shape[1], BLOCK):
        x, y = np.abs(a[:, k:k + BLOCK]), np.abs(b[k:k + BLOCK])
        largest = np.zeros_like(total)
        for i in range(x.shape[1]):
            np.maximum(largest, x[:, i:i + 1] * y[i], out=largest)
        total += 127 * 2.0 ** -13 * largest
    return total + (a.shape[1] / BLOCK + 2) * 2.0 ** -23 * (np.abs(a) @ np.abs(b))


def group_choice(scores, top_k, groups=1, top_groups=1, scoring="sigmoid", bias=None, best=2, normalize=True, scale=1.0):
    """(experts, weights) of every row."""
    tokens, experts = scores.shape
    size = experts // groups
    chosen, weights = np.zeros((tokens, top_k), dtype=np.int64), np.zeros((tokens, top_k))
    for t, s in enumerate(scores):
        masked = s == -np.inf
        if scoring == "sigmoid":
            with np.errstate(over="ignore"):
                p = np.where(s < 0, np.exp(np.minimum(s, 0)) / (1 + np.exp(np.minimum(s, 0))), 1 / (1 + np.exp(-np.maximum(s, 0))))
        else:
            p = np.zeros(experts) if masked.all() else np.exp(s - s.max()) / np.exp(s - s.max()).sum()
        c = np.where(masked, -np.inf, p if bias is None else p + bias)
        value = np.array([np.sort(c[g * size:(g + 1) * size])[::-1][:best].sum() for g in range(groups)])
        kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
        order = s if bias is None else c
        among = [e for g in sorted(kept) for e in range(g * size, (g + 1) * size)]
        chosen[t] = sorted(among, key=lambda e: (-order[e], e))[:top_k]
        w = p[chosen[t]]
        total = w.sum() if normalize else 1.0
        weights[t] = scale * w / total if total > 0 else 0.0
    return chosen, weights


def group_choice_gradient(scores, chosen, grad, scoring="sigmoid", normalize=True, scale=1.0):
    """d (sum grad * weights) / d scores for a given choice."""
    out = np.zeros(scores.shape)
    for t, s in enumerate(scores):
        if np.all(s == -np.inf):
            continue
        with np.errstate(over="ignore"):
            p = 1 / (1 + np.exp(-s)) if scoring == "sigmoid" else np.exp(s - s.max()) / np.exp(s - s.max()).sum()
        w = p[chosen[t]]
        total = w.sum() if normalize else 1.0
        if total == 0:
            continue
        dp = np.zeros(s.shape)
        dp[chosen[t]] = scale * (grad[t] - ((grad[t] * w).sum() / total if normalize else 0.0)) / total
        # (of a normalised row the sum of dp p is zero: what 64 bits leave of it would stand at experts that are not chosen)
        out[t] = dp * p * (1 - p) if scoring == "sigmoid" else p * (dp - (0.0 if normalize else (dp * p).sum()))
    return out
