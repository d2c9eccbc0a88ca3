"""8-bit floating point without a GPU: the oracle against torch's conversions, sizes, and what the C ABI refuses."""
import ctypes

import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import float8_oracle as F
from stk_amd.backend import _lib


def test_oracle_rounds_like_torch():
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = (codes[1:] + codes[:-1]) / 2
    v = torch.cat([codes, middle, middle * (1 - 2 ** -20), middle * (1 + 2 ** -20), torch.tensor([1e-30])])
    v = torch.cat([v, -v])
    assert np.array_equal(F.e4m3(v.numpy()), v.float().to(torch.float8_e4m3fn).double().numpy())


def test_powers():
    for most, e in ((448, 0), (448.0000001, 1), (224, -1), (225, 0), (1, -8), (2.0 ** -149, -126), (0, -126), (3.4e38, 120)):
        assert F.power_of(np.float64(most)) == 2.0 ** e, most


def test_sizes():
    lib = _lib.load()
    assert lib.stk_8bit_piece_bytes(2, 129, 65) == 2 * 8 * 2 * 2048
    assert lib.stk_8bit_scale_bytes(1, 129, 65, 0) == 128 * 4 and lib.stk_8bit_scale_bytes(3, 129, 300, 1) == 3 * 3 * 2 * 4
    assert lib.stk_8bit_row_bytes(3, 129) == 3 * 256 and lib.stk_8bit_exponent_bytes(3, 640) == 3 * 8
    for f in (lib.stk_8bit_piece_bytes, lib.stk_8bit_row_bytes, lib.stk_8bit_exponent_bytes):
        assert f(*[0] * len(f.argtypes)) == 0
    assert lib.stk_8bit_product_kernel(0, 1, 128, 128) == -1


@pytest.mark.parametrize("rows,experts", [(1, 1), (300, 1), (128, 64), (16384, 64), (5, 1024)])
def test_workspaces(rows, experts):
    lib = _lib.load()
    needs = lib.stk_matmul_8bit_workspace_bytes(rows, rows, experts, 1000, 512)
    assert needs == 0 if lib.stk_8bit_product_kernel(rows, experts, 1000, 512) < 5 else needs >= rows * 1032
    assert lib.stk_matmul_8bit_scatter_workspace_bytes(rows, 1, experts, 1000, 512) == needs
    assert lib.stk_matmul_8bit_scatter_workspace_bytes(rows * 2, 2, experts, 1000, 512) >= rows * 2 * 512 * 4


def _status(call):
    lib = _lib.load()
    return call(lib), lib.stk_last_error().decode()


def test_refusals_of_the_c_abi():
    """Nothing is launched: every call ends at its checks."""
    at = ctypes.c_void_p(4096)     # (never read)
    dims, unsupported, workspace = _lib.STK_ERR_DIMS, _lib.STK_ERR_UNSUPPORTED, _lib.STK_ERR_WORKSPACE
    bf16, f32 = _lib.STK_BF16, _lib.STK_F32
    odd = ctypes.c_void_p(4104)
    huge = 2 ** 31
    calls = [
        (dims, lambda l: l.stk_quantize_8bit(at, 0, 1, 1, 0, 128, 128, bf16, at, at, None, None, None)),
        (dims, lambda l: l.stk_quantize_8bit(None, 0, 1, 1, 1, 128, 128, bf16, at, at, None, None, None)),
        (dims, lambda l: l.stk_quantize_8bit(at, 0, 1, 1, 1, 128, 128, bf16, at, at, at, None, None)),
        (unsupported, lambda l: l.stk_quantize_8bit(at, 0, 1, 1, 1, 128, 128, 7, at, at, None, None, None)),
        (unsupported, lambda l: l.stk_quantize_8bit(at, 0, 1, 1, 1, huge, 128, bf16, at, at, None, None, None)),
        (unsupported, lambda l: l.stk_quantize_8bit(at, 0, 1, 1, 1, 128, 128, bf16, odd, at, None, None, None)),
        (dims, lambda l: l.stk_pack_8bit(at, None, 0, 1, 128, 128, at, at, None)),
        (dims, lambda l: l.stk_dequantize_8bit(at, at, 0, 1, 0, 128, at, bf16, None)),
        (dims, lambda l: l.stk_quantize_rows_8bit(at, -1, 128, 128, bf16, at, at, None, None, 0, None)),
        (dims, lambda l: l.stk_quantize_rows_8bit(at, 4, 128, 128, bf16, None, None, None, None, 0, None)),
        (dims, lambda l: l.stk_quantize_rows_8bit(at, 4, 128, 128, bf16, at, None, None, None, 0, None)),
        (unsupported, lambda l: l.stk_quantize_rows_8bit(at, 65536 * 128, 128, 128, bf16, None, None, at, at, 0, None)),
        (unsupported, lambda l: l.stk_matmul_8bit(at, 4, 128, at, at, 0, 128, 128, at, 128, 0, f32, None, 0, None)),
        (unsupported, lambda l: l.stk_matmul_8bit(at, 4, 128, odd, at, 0, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (unsupported, lambda l: l.stk_matmul_8bit(at, 4, 128, at, at, 0, 128, 128, at, 128, 5, bf16, None, 0, None)),
        (dims, lambda l: l.stk_matmul_8bit(at, 4, 128, at, at, 0, 128, 128, at, 127, 0, bf16, None, 0, None)),
        (dims, lambda l: l.stk_matmul_8bit(at, -4, 128, at, at, 0, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (dims, lambda l: l.stk_matmul_8bit(at, 4, 128, None, at, 0, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (workspace, lambda l: l.stk_matmul_8bit(at, 400000, 128, at, at, 0, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (workspace, lambda l: l.stk_matmul_8bit(at, 400000, 128, at, at, 0, 128, 128, at, 128, 0, bf16, odd, 1 << 30, None)),
        (dims, lambda l: l.stk_gather_matmul_8bit(at, 4, 128, None, at, 1, at, at, 0, 2, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (dims, lambda l: l.stk_gather_matmul_8bit(at, huge, 128, at, at, 2, at, at, 0, 2, 128, 128, at, 128, 0, bf16, None, 0, None)),
        (workspace, lambda l: l.stk_matmul_8bit_scatter(at, 128, at, at, 2, 4, None, at, at, 0, 2, 128, 128, at, 128, bf16, None, 0, None)),
        (dims, lambda l: l.stk_linear_8bit(at, at, 128, None, at, at, 2, 128, 128, at, 128, bf16, None)),
        (dims, lambda l: l.stk_linear_8bit(at, None, 128, None, at, at, 1, 128, 128, at, 128, bf16, None)),
        (unsupported, lambda l: l.stk_linear_8bit(at, at, 128, None, at, at, 1, 2 ** 23 + 1, 128, at, 128, bf16, None)),
        (unsupported, lambda l: l.stk_weight_gradient_8bit(at, at, at, at, 2 ** 23 + 1, None, 1, 128, 128, at, bf16, None)),
        (dims, lambda l: l.stk_weight_gradient_8bit(at, at, at, at, 0, None, 1, 128, 128, at, bf16, None)),
        (dims, lambda l: l.stk_weight_gradient_8bit(at, at, at, at, 128, None, 2, 128, 128, at, bf16, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 30, 30, 4, 2, 1, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 4, 5, 1, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 4, 1, 1, 9, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 4, 1, 3, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 32, 1, 2, 1, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 4, 1, 1, 2, 0, None, 0, float("nan"), at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(at, 4, 32, 32, 4, 1, 1, 2, 0, None, 0, 0.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts(None, 4, 32, 32, 4, 1, 1, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (unsupported, lambda l: l.stk_group_top_experts(at, 4, 1040, 1040, 4, 1, 1, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (unsupported, lambda l: l.stk_group_top_experts(at, 4, 320, 320, 80, 1, 1, 2, 0, None, 0, 1.0, at, at, f32, None)),
        (unsupported, lambda l: l.stk_group_top_experts(at, 4, 320, 320, 4, 4, 1, 33, 0, None, 0, 1.0, at, at, f32, None)),
        (dims, lambda l: l.stk_group_top_experts_backward(at, 32, at, at, None, 4, 32, 2, 0, 0, 1.0, at, 32, f32, None)),
        (dims, lambda l: l.stk_group_top_experts_backward(at, 32, at, at, at, 4, 32, 2, 0, 0, 1.0, at, 31, f32, None)),
    ]
    for n, (want, call) in enumerate(calls):
        got, text = _status(call)
        assert got == want and text, (n, got, text)


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(128, 128, dtype=torch.bfloat16)
    for call in (lambda: stk.ops.linear_8bit(x, w), lambda: stk.ops.quantize_8bit(w), lambda: stk.ops.group_top_experts(torch.zeros(4, 8), 2)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        stk.ops.group_top_experts(torch.zeros(4, 8), 2, scoring="tanh")
