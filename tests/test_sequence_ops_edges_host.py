"""Refusals of the sequence operators at the ends of their numbers (no GPU needed)."""

import ctypes as C
import struct

import pytest

import ppocr_b200 as P
import test_sequence_ops_host as ops

gpu = ops.gpu   # the stand-in handle; nothing below reaches a device


@pytest.mark.parametrize("call", [ops.packed, ops.cached])
@pytest.mark.parametrize("scale", [1e-50, 5e-324, 2.0 ** -150, 1e-46])
def test_a_scale_that_is_zero_in_fp32_is_refused(gpu, call, scale):
    """0 is the library's word for the default, d^-1/2."""
    assert struct.unpack("f", struct.pack("f", scale))[0] == 0
    with pytest.raises(P.InvalidInput, match="scale"):
        call(gpu, scale=scale)


@pytest.mark.parametrize("call", [ops.packed, ops.cached])
@pytest.mark.parametrize("scale", [1.0000001 * 2.0 ** -150, 2.0 ** -149, 1e-30])
def test_the_smallest_scales_pass_the_checks(gpu, call, scale):
    assert C.c_float(scale).value > 0
    if P.gpu_count() > 0:
        pytest.skip("the stand-in handle must not reach a device")
    with pytest.raises(P.GpuError):
        call(gpu, scale=scale)
