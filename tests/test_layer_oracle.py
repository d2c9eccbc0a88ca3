"""CPU tier of the operators around the products: the 64-bit definitions are pinned by torch's own functions and by
differences, and the entry points' refusals are those that need no GPU."""
import ctypes

import numpy as np
import pytest
import torch

import stk_amd as stk
from oracle import layer_oracle as L
from stk_amd.backend import _lib


@pytest.mark.parametrize("rows,size", [(1, 1), (3, 2), (4, 7), (5, 33)])
def test_layer_norm_definition_is_torchs(rows, size):
    g = torch.Generator().manual_seed(size)
    x, dy = (torch.randn(rows, size, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(size, generator=g, dtype=torch.float64) for _ in range(2))
    for t in (x, w, b):
        t.requires_grad_(True)
    y = torch.nn.functional.layer_norm(x, (size,), w, b, 1e-5)
    want = torch.autograd.grad(y, (x, w, b), dy)
    got = L.layer_norm_gradients(dy, x.detach(), w.detach())
    np.testing.assert_allclose(L.layer_norm(x.detach(), w.detach(), b.detach())[0], y.detach(), rtol=1e-12, atol=1e-12)
    for a, c in zip(got, want):
        np.testing.assert_allclose(a, c, rtol=1e-9, atol=1e-9)


def test_layer_norm_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, w, dy = rng.normal(size=(2, 5)), rng.normal(size=5), rng.normal(size=(2, 5))
    dx, dw, db = L.layer_norm_gradients(dy, x, w)
    f = lambda x, w, b: (L.layer_norm(x, w, b)[0] * dy).sum()
    h = 1e-6
    for at in np.ndindex(2, 5):
        step = np.zeros((2, 5))
        step[at] = h
        assert abs((f(x + step, w, None) - f(x - step, w, None)) / (2 * h) - dx[at]) < 1e-7
    for i in range(5):
        step = np.zeros(5)
        step[i] = h
        assert abs((f(x, w + step, None) - f(x, w - step, None)) / (2 * h) - dw[i]) < 1e-7
        assert abs((f(x, w, step) - f(x, w, -step)) / (2 * h) - db[i]) < 1e-7


@pytest.mark.parametrize("normalize", [False, True])
def test_top_experts_definition(normalize):
    g = torch.Generator().manual_seed(2)
    s = torch.randn(6, 9, generator=g, dtype=torch.float64).requires_grad_(True)
    dw = torch.randn(6, 3, generator=g, dtype=torch.float64)
    p = torch.softmax(s, dim=1)
    want, idx = p.topk(3, dim=1)
    if normalize:
        want = want / want.sum(dim=1, keepdim=True)
    chosen, weights = L.top_experts(s.detach(), 3, normalize)
    assert np.array_equal(chosen, idx)
    np.testing.assert_allclose(weights, want.detach(), rtol=1e-12)
    np.testing.assert_allclose(L.top_experts_gradient(s.detach(), 3, dw, normalize), torch.autograd.grad(want, s, dw)[0], rtol=1e-9, atol=1e-12)


def test_top_experts_definition_of_ties_masks_and_nan():
    inf, nan = np.inf, np.nan
    s = np.array([[1., 2., 2., 0.], [-inf, -inf, 3., -inf], [-inf] * 4, [0., nan, 9., 1.], [5., inf, 1., 0.], [0., -0., 0., -0.]])
    chosen, weights = L.top_experts(s, 2)
    assert chosen.tolist() == [[1, 2], [2, 0], [0, 1], [1, 2], [1, 0], [0, 1]]
    assert weights[1].tolist() == [1., 0.] and weights[2].tolist() == [0., 0.]
    assert np.isnan(weights[3]).all() and np.isnan(weights[4]).all()
    assert L.top_experts(s, 2, True)[1][1].tolist() == [1., 0.]
    assert not L.top_experts_gradient(s[2:3], 2, np.ones((1, 2))).any()


def test_products_of_4bit_weights_definition():
    rng = np.random.default_rng(3)
    codes, scales, offsets = rng.integers(0, 16, (2, 6, 4)).astype(np.uint8), rng.random((2, 2, 4)), rng.random((2, 2, 4))
    w, wo = L.weights4(codes, scales, 4), L.weights4(codes, scales, 4, offsets)
    for e, i, o in np.ndindex(2, 6, 4):
        assert w[e, i, o] == scales[e, i // 4, o] * (int(codes[e, i, o]) - 8)
        assert wo[e, i, o] == scales[e, i // 4, o] * codes[e, i, o] + offsets[e, i // 4, o]
    # three tokens with two choices each: slots of expert 0: 1, 2; of expert 1: 0, 3, 4, 5
    indices, bins = np.array([1, 2, 0, 3, 4, 5]), np.array([2, 6])
    x, by = rng.random((3, 6)), rng.random(6)
    h = L.gather_matmul(x, indices, bins, 2, w)
    np.testing.assert_allclose(h[1], x[1] @ w[0])
    np.testing.assert_allclose(h[4], x[2] @ w[1])
    y = L.matmul_scatter(rng.random((6, 6)) * 0 + np.arange(6)[:, None], indices, bins, 2, w, by)
    np.testing.assert_allclose(y[0], by[0] * 2 * w[1].sum(axis=0) + by[1] * 0 * w[0].sum(axis=0))


# ---------------------------------------------------------------------------------------------------- refusals
def _bad(status, code, text):
    assert status == code, (status, _lib.load().stk_last_error())
    assert text in _lib.load().stk_last_error().decode()


def test_abi_refusals_of_layer_norm():
    lib, one = _lib.load(), ctypes.c_void_p(256)      # (an address that no refused call touches)
    _bad(lib.stk_layer_norm(one, 4, 0, 8, None, None, 1e-5, one, 8, None, None, _lib.STK_F32, _lib.STK_F32, None), _lib.STK_ERR_DIMS, "stk_layer_norm")
    _bad(lib.stk_layer_norm(one, 4, 8, 8, None, None, 1e-5, one, 8, None, None, 7, 7, None), _lib.STK_ERR_UNSUPPORTED, "dtype 7")
    _bad(lib.stk_layer_norm(one, 4, 8, 8, one, None, 1e-5, one, 8, None, None, _lib.STK_BF16, _lib.STK_F16, None), _lib.STK_ERR_UNSUPPORTED, "float32")
    _bad(lib.stk_layer_norm(one, 4, 8, 8, None, None, 1e-5, one, 7, None, None, _lib.STK_F32, _lib.STK_F32, None), _lib.STK_ERR_DIMS, "strides")
    _bad(lib.stk_layer_norm(one, 4, 8, 8, None, None, 1e-5, one, 8, one, None, _lib.STK_F32, _lib.STK_F32, None), _lib.STK_ERR_DIMS, "missing pointer")
    assert lib.stk_layer_norm(None, 0, 8, 8, None, None, 1e-5, None, 8, None, None, _lib.STK_F32, _lib.STK_F32, None) == _lib.STK_OK
    _bad(lib.stk_layer_norm_backward(one, 8, one, 8, one, one, None, 4, 8, one, 8, one, None, _lib.STK_F32, _lib.STK_F32, None, 0, None), _lib.STK_ERR_WORKSPACE,
         "workspace")
    _bad(lib.stk_layer_norm_backward(one, 8, one, 8, None, None, None, 4, 8, one, 8, None, None, _lib.STK_F32, _lib.STK_F32, None, 0, None), _lib.STK_ERR_DIMS,
         "missing pointer")


def test_abi_refusals_of_top_experts():
    lib, one = _lib.load(), ctypes.c_void_p(256)
    call = lambda experts, k, dtype=_lib.STK_F32, scores=one: lib.stk_top_experts(scores, 4, experts, experts, k, 0, one, one, dtype, None)
    _bad(call(4, 5), _lib.STK_ERR_DIMS, "top 5 of 4")
    _bad(call(4, 0), _lib.STK_ERR_DIMS, "top 0")
    _bad(call(1025, 1), _lib.STK_ERR_UNSUPPORTED, "1024 experts")
    _bad(call(100, 65), _lib.STK_ERR_UNSUPPORTED, "the top 64")
    _bad(call(4, 2, 3), _lib.STK_ERR_UNSUPPORTED, "dtype 3")
    _bad(call(4, 2, scores=None), _lib.STK_ERR_DIMS, "missing pointer")
    _bad(lib.stk_top_experts_backward(None, 4, one, one, one, 4, 4, 2, 0, one, 4, _lib.STK_F32, None), _lib.STK_ERR_DIMS, "missing pointer")
    _bad(lib.stk_top_experts_backward(one, 4, one, one, one, 4, 4, 2, 0, one, 3, _lib.STK_F32, None), _lib.STK_ERR_DIMS, "strides")


def test_abi_refusals_and_sizes_of_4bit_weights():
    lib, one = _lib.load(), ctypes.c_void_p(256)
    assert lib.stk_4bit_packed_bytes(3, 129, 17) == 3 * 2 * 2 * 1024 and lib.stk_4bit_packed_bytes(1, 0, 17) == 0
    # whole pieces of 128 inputs, whole blocks of the groups of a piece, 16 outputs
    assert lib.stk_4bit_scales(3, 129, 17, 32) == 3 * 8 * 32 and lib.stk_4bit_scales(1, 128, 16, 256) == 16
    mm = lambda group=128, dtype=_lib.STK_BF16, act=0, x=one, out_stride=16, packed=one: lib.stk_matmul_4bit(
        x, 4, 128, packed, one, None, 128, 16, group, one, out_stride, act, dtype, None)
    _bad(mm(group=48), _lib.STK_ERR_UNSUPPORTED, "groups of 32, 64 or a multiple of 128")
    _bad(mm(group=0), _lib.STK_ERR_DIMS, "groups of 0")
    _bad(mm(dtype=_lib.STK_F32), _lib.STK_ERR_UNSUPPORTED, "dtype 2")
    _bad(mm(act=5), _lib.STK_ERR_UNSUPPORTED, "activation 5")
    _bad(mm(x=None), _lib.STK_ERR_DIMS, "missing pointer")
    _bad(mm(out_stride=15), _lib.STK_ERR_DIMS, "strides")
    _bad(mm(packed=ctypes.c_void_p(264)), _lib.STK_ERR_UNSUPPORTED, "multiples of 16 bytes")
    _bad(lib.stk_gather_matmul_4bit(one, 4, 128, None, one, 2, one, one, None, 4, 128, 16, 128, one, 16, 0, _lib.STK_BF16, None), _lib.STK_ERR_DIMS,
         "missing pointer")
    _bad(lib.stk_gather_matmul_4bit(one, 4, 128, one, one, 0, one, one, None, 4, 128, 16, 128, one, 16, 0, _lib.STK_BF16, None), _lib.STK_ERR_DIMS, "top_k 0")
    _bad(lib.stk_matmul_4bit_scatter(one, 128, one, one, 2, 4, None, one, one, None, 4, 128, 16, 128, one, 16, _lib.STK_BF16, None, 0, None), _lib.STK_ERR_WORKSPACE,
         "workspace")
    _bad(lib.stk_pack_4bit(one, one, one, 1, 128, 16, 128, one, one, None, None), _lib.STK_ERR_DIMS, "missing pointer")
    _bad(lib.stk_quantize_4bit(one, 1, 1, 1, 1, 128, 16, 128, one, one, None, _lib.STK_F16, _lib.STK_BF16, None), _lib.STK_ERR_UNSUPPORTED, "float32")


def test_host_tensors_are_refused():
    x = torch.zeros(4, 128)
    codes, scales = torch.zeros(128, 16, dtype=torch.uint8), torch.ones(1, 16, dtype=torch.bfloat16)
    for call in (lambda: stk.ops.layer_norm(x), lambda: stk.ops.top_experts(x, 2), lambda: stk.ops.pack_4bit(codes, scales, 128),
                 lambda: stk.ops.quantize_4bit(x, dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError, match="ROCm GPU only"):
            call()
