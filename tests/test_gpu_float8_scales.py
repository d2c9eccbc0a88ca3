"""8-bit weights with fp32 scales far from 1, met by rows far from 1 on the other side.

Powers of two do not change the bits of a product (test_gpu_float8.py): where the product of a row's scale and a weight's is what it was, so is the result,
and whole numbers times powers of two have exact sums.
"""
import pytest
import torch

import stk_amd as stk
from stk_amd.backend import _lib
from tests.test_gpu_float8 import DEV, _whole

pytestmark = pytest.mark.gpu
# a size for each kernel of the rule
SIZES = [(1, 300, 96), (20, 256, 4096), (20, 1104, 8192), (40, 640, 4096), (16, 300, 70000), (1000, 520, 513), (200, 513, 8200), (1000, 256, 4100), (3500, 256, 3500)]


def _packed(codes, scales):
    return stk.ops.pack_8bit(codes.to(torch.float8_e4m3fn).to(DEV), scales.to(DEV))


def test_every_kernel_is_reached():
    lib = _lib.load()
    assert {lib.stk_8bit_product_kernel(r, 1, i, o) for r, i, o in SIZES} >= set(range(9))


@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_same_bits(rows, inputs, outputs):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, inputs, generator=g).bfloat16().to(DEV)
    codes = (torch.randn(inputs, outputs, generator=g) * 80).clamp(-448, 448)
    scales = (torch.rand((inputs + 127) // 128, (outputs + 127) // 128, generator=g) + 0.5)
    scales[::2] *= -1
    want = stk.ops.matmul_8bit(x, _packed(codes, scales))
    assert torch.isfinite(want).all()
    for power in (120, 90, -90):
        assert torch.equal(stk.ops.matmul_8bit(x * 2.0 ** power, _packed(codes, scales * 2.0 ** -power)), want), power


@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
@pytest.mark.parametrize("of_rows,of_weights", [(118, -60), (112, -130), (112, -145), (-120, 122), (-126, 127)])
def test_whole_numbers(rows, inputs, outputs, of_rows, of_weights):
    """Also scales below the normal numbers of fp32."""
    g = torch.Generator().manual_seed(outputs)
    x, codes = _whole((rows, inputs), g), _whole((inputs, outputs), g)
    scales = torch.full(((inputs + 127) // 128, (outputs + 127) // 128), 2.0 ** of_weights)
    want = ((x.double() @ codes.double()) * 2.0 ** (of_rows + of_weights)).float().bfloat16()
    got = stk.ops.matmul_8bit((x.double() * 2.0 ** of_rows).bfloat16().to(DEV), _packed(codes, scales))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_blocks_of_scale_zero_and_infinity(rows, inputs, outputs):
    """A block of scale 0 adds nothing to rows of any size; one of infinity leaves nothing finite."""
    g = torch.Generator().manual_seed(inputs)
    x, codes = torch.randn(rows, inputs, generator=g).abs().bfloat16() * 2.0 ** 119, _whole((inputs, outputs), g).abs() + 1
    scales = torch.full(((inputs + 127) // 128, (outputs + 127) // 128), 2.0 ** -60)
    first = stk.ops.matmul_8bit(x[:, :128].contiguous().to(DEV), _packed(codes[:128], scales[:1]))
    zero = scales.clone()
    zero[1:] = 0.0
    assert torch.equal(stk.ops.matmul_8bit(x.to(DEV), _packed(codes, zero)), first)
    zero[-1] = float("inf")
    assert not torch.isfinite(stk.ops.matmul_8bit(x.to(DEV), _packed(codes, zero))).any()
