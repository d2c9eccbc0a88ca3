"""CPU tier of the 4-bit weights: what the library says about their sizes and about the kernels that the tests reach."""
import pytest

from stk_amd.backend import _lib
from tests import _weights4_cases as cases


@pytest.mark.parametrize("inputs", [1, 128, 129, 4096, 5000])
def test_groups_beyond_the_inputs_are_one_group(inputs):
    """Whatever multiple of 128 it is, up to the largest that 64 bits hold: the scales of one group of whole pieces."""
    lib = _lib.load()
    whole = (inputs + 127) // 128 * 128
    want = lib.stk_4bit_scales(3, inputs, 40, whole)
    assert want == 3 * 48
    for group in (whole, whole + 128, 1 << 26, 1 << 31, 1 << 38, 1 << 39, (1 << 39) + 128, 1 << 62, (1 << 63) - 128):
        assert lib.stk_4bit_scales(3, inputs, 40, group) == want, group


@pytest.mark.parametrize("kernel", cases.KERNELS)
def test_the_sizes_of_the_gpu_tests_take_every_kernel(kernel):
    """tests/test_gpu_weights4_kernels.py runs these at every class of groups, with and without offsets, in both types."""
    lib, number = _lib.load(), cases.KERNELS.index(kernel)
    tokens, experts, top_k, inputs, outputs = cases.ROUTED[kernel]
    assert lib.stk_4bit_product_kernel(tokens * top_k, experts, inputs, outputs, inputs % 8 == 0) == number
    rows, inputs, outputs = cases.PLAIN[kernel]
    assert lib.stk_4bit_product_kernel(rows, 1, inputs, outputs, inputs % 8 == 0) == number
    for inputs in (cases.ROUTED[kernel][3], cases.PLAIN[kernel][1]):
        assert inputs % 128 and inputs > max(cases.GROUPS)


def test_the_rule_has_no_other_kernel():
    lib = _lib.load()
    seen = {lib.stk_4bit_product_kernel(rows, experts, inputs, outputs, whole)
            for rows in (1, 2, 7, 16, 40, 64, 200, 513, 2000, 16384, 100000) for experts in (1, 2, 8, 64, 1000) for inputs in (1, 128, 1000, 4096, 20000)
            for outputs in (1, 100, 1024, 5000, 70000) for whole in (0, 1)}
    assert seen == set(range(len(cases.KERNELS))) == set(map(cases.KERNELS.index, cases.ROUTED)) == set(map(cases.KERNELS.index, cases.PLAIN))
    assert lib.stk_4bit_product_kernel(0, 1, 1, 1, 1) == -1 and lib.stk_4bit_product_kernel(1, 0, 1, 1, 1) == -1
