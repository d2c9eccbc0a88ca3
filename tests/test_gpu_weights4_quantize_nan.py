"""GPU: weights that have no finite 4-bit form are quantized to NaN, not to a number that looks like one of the others."""
import pytest
import torch

import stk_amd as stk

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _groups(dtype, to, affine):
    """(name, weights of one group of 32) that have no finite form."""
    inf, nan = float("inf"), float("nan")
    some = torch.linspace(-1, 1, 32)
    yield "a NaN", torch.where(torch.arange(32) == 5, nan, some)
    yield "NaN only", torch.full((32,), nan)
    yield "+infinity", torch.where(torch.arange(32) == 31, inf, some)
    yield "-infinity", torch.where(torch.arange(32) == 0, -inf, some)
    yield "both", torch.where(torch.arange(32) == 0, -inf, torch.where(torch.arange(32) == 9, inf, some))
    yield "infinity and NaN", torch.where(torch.arange(32) == 0, nan, torch.where(torch.arange(32) == 9, inf, some))
    if dtype == torch.float32:
        big = 1e6 if to == torch.float16 else 3.4e38     # beyond the largest finite number of the scales' type, once divided
        yield "too large for the scale", torch.where(torch.arange(32) % 2 == 0, big * (1 if to == torch.float16 else 1.0), -big * 1.0)
        if affine and to == torch.float16:
            yield "too large for the offset", torch.where(torch.arange(32) == 3, -70000.0, 0.0)
            yield "all alike and too large", torch.full((32,), 1e6)


@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("dtype,to", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
def test_weights_without_a_finite_form_become_nan(dtype, to, affine):
    """Every weight of their group; the others are those of the clean matrix."""
    g = torch.Generator().manual_seed(4)
    clean = (torch.randn(100, 16, generator=g) * 0.1).to(dtype)
    x = torch.randn(5, 100, generator=g).to(to).to(DEV)
    near = stk.ops.quantize_4bit(clean.to(DEV), 32, offsets=affine, dtype=to)
    want, y = stk.ops.dequantize_4bit(near), stk.ops.matmul_4bit(x, near, "relu")
    for name, group in _groups(dtype, to, affine):
        if name == "too large for the scale" and to == torch.bfloat16 and not affine:
            continue      # (a seventh of the largest float32 number is a bfloat16 one)
        w = clean.clone()
        w[32:64, 7] = group.to(dtype)
        q = stk.ops.quantize_4bit(w.to(DEV), 32, offsets=affine, dtype=to)
        got = stk.ops.dequantize_4bit(q)
        hit = torch.zeros(100, 16, dtype=torch.bool, device=DEV)
        hit[32:64, 7] = True
        assert torch.isnan(got[hit]).all(), name
        assert torch.equal(got[~hit], want[~hit]), name
        out = stk.ops.matmul_4bit(x, q, "relu")
        others = [o for o in range(16) if o != 7]
        assert torch.isnan(out[:, 7]).all() and torch.equal(out[:, others], y[:, others]), name
