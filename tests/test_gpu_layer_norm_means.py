"""GPU: the mean of a row of equal values is that value, so that such a row has no deviation and its result is the bias, to the last bit.

Why that can be asked for: the mean is the row's first value plus the mean of the differences from it, which are 0 here, exactly, in whatever
order they are added up."""
import pytest
import torch

import stk_amd as stk
from stk_amd.backend import hip_kernels
from tests.test_gpu_layer_norm import _run

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [1, 3, 7, 41, 47, 100, 128, 500, 1000, 1024, 1151, 2000, 3001, 4096, 7168, 8192, 12345, 16384, 20001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_constant_rows(size, dtype):
    values = torch.tensor([1000.0, 0.1, -3.7, 1.0 / 3.0, 60000.0, 0.0, 1e-3, 2.0]).to(dtype)
    x = values.unsqueeze(1).expand(8, size).contiguous().to(DEV)
    g = torch.Generator().manual_seed(size)
    w, b, dy = torch.randn(size, generator=g).to(dtype).to(DEV), torch.randn(size, generator=g).to(dtype).to(DEV), torch.randn(8, size, generator=g).to(dtype).to(DEV)
    assert not stk.ops.layer_norm(x).any()
    y, grads = _run(x, w, b, dy)
    assert torch.equal(y, b.expand(8, size))
    assert not grads[1].any()
    _, statistics = hip_kernels.layer_norm(x, None, None, 1e-5, with_statistics=True)
    assert torch.equal(statistics[0], x[:, 0].float())
