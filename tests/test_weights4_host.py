"""CPU tier of the 4-bit weights: what the library says about their sizes."""
import pytest

from stk_amd.backend import _lib


@pytest.mark.parametrize("inputs", [1, 128, 129, 4096, 5000])
def test_groups_beyond_the_inputs_are_one_group(inputs):
    """Whatever multiple of 128 it is, up to the largest that 64 bits hold: the scales of one group of whole pieces."""
    lib = _lib.load()
    whole = (inputs + 127) // 128 * 128
    want = lib.stk_4bit_scales(3, inputs, 40, whole)
    assert want == 3 * 48
    for group in (whole, whole + 128, 1 << 26, 1 << 31, 1 << 38, 1 << 39, (1 << 39) + 128, 1 << 62, (1 << 63) - 128):
        assert lib.stk_4bit_scales(3, inputs, 40, group) == want, group
