"""GPU: what is not a number stays visible in the products with 4-bit weights, whatever the activation, and what is a number stays one."""
import pytest
import torch

import stk_amd as stk
from oracle import layer_oracle as L
from tests.test_gpu_weights4 import ACT, HALF, _check, _n64, _pack, _slack, _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
# few rows, rows through registers and rows in whole 16-byte pieces
SIZES = [(2, 300, 40), (100, 301, 4100), (200, 304, 1920), (700, 304, 6688)]


@pytest.mark.parametrize("activation", list(ACT))
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_rows_with_infinities_and_nan_are_nan_behind_every_activation(rows, inputs, outputs, dtype, activation):
    codes, scales, offsets = _weights((inputs, outputs), 32, True, dtype, 9)
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).to(dtype).to(DEV)
    bad = x.clone()
    bad[0, 7], bad[rows - 1, inputs - 1] = -float("inf"), float("nan")
    for w in (_pack(codes, scales, None, 32), _pack(codes, scales, offsets, 32)):
        want, got = stk.ops.matmul_4bit(x, w, activation), stk.ops.matmul_4bit(bad, w, activation)
        assert torch.isfinite(want).all()
        assert torch.isnan(got[[0, rows - 1]]).all()
        assert torch.equal(got[1:rows - 1], want[1:rows - 1])


@pytest.mark.parametrize("activation", list(ACT))
def test_routed_rows_with_infinities_and_nan(activation):
    codes, scales, _ = _weights((4, 200, 48), 64, False, torch.float16, 3)
    w = _pack(codes, scales, None, 64)
    g = torch.Generator().manual_seed(1)
    route = stk.ops.route(torch.randint(0, 4, (30, 2), generator=g, dtype=torch.int32).to(DEV), 4, 1)
    x = torch.randn(30, 200, generator=g).half().to(DEV)
    want = stk.ops.gather_matmul_4bit(x, route, w, activation)
    bad = x.clone()
    bad[3, 0], bad[20, 199] = float("inf"), float("nan")
    got = stk.ops.gather_matmul_4bit(bad, route, w, activation)
    token = route.indices.long() // 2
    hit = (token == 3) | (token == 20)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])
    # and on the way back, where the token's sum meets it
    y = stk.ops.matmul_4bit_scatter(bad[token], route, w)
    hit = torch.zeros(30, dtype=torch.bool, device=DEV)
    hit[[3, 20]] = True
    assert torch.isnan(y[hit]).all() and torch.isfinite(y[~hit]).all()


@pytest.mark.parametrize("affine", [False, True])
def test_large_rows_are_numbers(affine):
    """Sums of |x| up to 2^123 do not overflow on their way (the codes are multiplied as numbers up to 31)."""
    codes, scales, offsets = _weights((256, 64), 64, affine, torch.bfloat16, 5)
    x = torch.randn(9, 256, generator=torch.Generator().manual_seed(2)).bfloat16()
    x[1, 3], x[2, 255], x[5] = 2.0 ** 122, -2.0 ** 122, 2.0 ** 114
    got = stk.ops.matmul_4bit(x.to(DEV), _pack(codes, scales, offsets, 64))
    _check(got, _n64(x) @ L.weights4(codes.numpy(), _n64(scales), 64, _n64(offsets)), _slack(x, codes, scales, offsets, 64), torch.bfloat16)
