"""GPU: group sizes beyond the inputs mean one group of them all, up to the largest multiple of 128 that 64 bits hold."""
import pytest
import torch

import stk_amd as stk
from tests.test_gpu_weights4 import _weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs", [(3, 300, 40), (160, 300, 640), (200, 304, 1920), (200, 301, 1920), (3, 3200, 40), (16, 128, 40), (2, 5, 17)])
def test_groups_beyond_the_inputs(rows, inputs, outputs, affine):
    whole = (inputs + 127) // 128 * 128
    codes, scales, offsets = (None if t is None else t.to(DEV) for t in _weights((inputs, outputs), whole, affine, torch.bfloat16, rows))
    x = torch.randn(rows, inputs, generator=torch.Generator().manual_seed(rows)).bfloat16().to(DEV)
    w = stk.ops.pack_4bit(codes, scales, whole, offsets)
    want, dense = stk.ops.matmul_4bit(x, w), stk.ops.dequantize_4bit(w)
    for group in (whole + 128, 1 << 31, 1 << 39, (1 << 39) + 128, (1 << 63) - 128):
        far = stk.ops.pack_4bit(codes, scales, group, offsets)
        assert torch.equal(far.packed, w.packed) and torch.equal(far.scales, w.scales)
        assert torch.equal(stk.ops.dequantize_4bit(far), dense)
        assert torch.equal(stk.ops.matmul_4bit(x, far), want)
        again = stk.ops.quantize_4bit(dense, group, offsets=affine)
        near = stk.ops.quantize_4bit(dense, whole, offsets=affine)
        assert torch.equal(again.packed, near.packed) and torch.equal(again.scales, near.scales)


def test_routed_groups_beyond_the_inputs():
    codes, scales, _ = (None if t is None else t.to(DEV) for t in _weights((4, 200, 48), 256, False, torch.bfloat16, 7))
    g = torch.Generator().manual_seed(3)
    route = stk.ops.route(torch.randint(0, 4, (50, 2), generator=g, dtype=torch.int32).to(DEV), 4, 1)
    x, h = torch.randn(50, 200, generator=g).bfloat16().to(DEV), torch.randn(100, 200, generator=g).bfloat16().to(DEV)
    near, far = stk.ops.pack_4bit(codes, scales, 256), stk.ops.pack_4bit(codes, scales, 1 << 39)
    assert torch.equal(stk.ops.gather_matmul_4bit(x, route, far), stk.ops.gather_matmul_4bit(x, route, near))
    assert torch.equal(stk.ops.matmul_4bit_scatter(h, route, far), stk.ops.matmul_4bit_scatter(h, route, near))
