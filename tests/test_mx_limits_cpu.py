"""Refusals of the MXFP4 operators that need no GPU: nothing is read or launched."""
import pytest

import ruquant_amd as rq

PTR = 1 << 20   # an aligned address that nothing is read from: the calls are refused first
ARGUMENT = -3


@pytest.mark.parametrize("dtype,off", [(0, 1), (0, 2), (1, 1), (2, 1), (2, 3)])
def test_quantizer_and_dequantizer_refuse_elements_at_broken_addresses(dtype, off):
    L = rq.load_library()
    assert L.rq_mx4_quantize(dtype, PTR + off, 64, 1, 64, PTR, PTR, None) == ARGUMENT
    assert L.rq_mx4_dequantize(dtype, PTR, PTR, 1, 64, PTR + off, 64, None) == ARGUMENT
    assert L.rq_mx4_quantize(dtype, PTR, 64, 1, 64, PTR + 2, PTR, None) == ARGUMENT
    assert L.rq_mx4_dequantize(dtype, PTR + 2, PTR, 1, 64, PTR, 64, None) == ARGUMENT
