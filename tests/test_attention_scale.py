"""The scale of the attention as fp32 bits, on the CPU."""
import struct

import pytest

from lynnreal_omni_amd import attention as A


@pytest.mark.parametrize("scale", [1e39, 1e308, float("inf"), -1.0, 0.0, float("nan")])
def test_scales_outside_fp32_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        A._scale_bits(scale)


@pytest.mark.parametrize("scale", [1e-45, 2.0 ** -126, 0.125, 3e38])
def test_scales_of_fp32_are_kept(scale):
    assert A._scale_bits(scale) == struct.unpack("i", struct.pack("f", scale))[0]
