"""Pointers that are not aligned to their elements are refused by the 8-bit and
expert entry points before any CUDA call (the kernels would read them)."""

import ctypes

import pytest

from test_fp8 import P, lib, matrix  # noqa: F401  (fixture)
from tensorpack_b200 import _lib

TEXT = b"aligned to"


def refused(lib, rc):
    assert rc == _lib.MTC_ERR_INVALID and TEXT in lib.mtc_last_error(), (rc, lib.mtc_last_error())


@pytest.mark.parametrize("t,off", [(0, 2), (0, 1), (1, 1), (2, 1)])
def test_activations_and_outputs(lib, t, off):
    w = matrix()
    gate, down = matrix(E=4, K=256, N=128), matrix(E=4, K=128, N=256, ldk=128)
    for x, y in ((P + off, P), (P, P + off)):
        refused(lib, lib.mtc_fp8_gemm(ctypes.byref(w), x, t, 1, 256, y, t, 128, None, 0, None, None, None))
        refused(lib, lib.mtc_experts_forward(ctypes.byref(gate), ctypes.byref(gate), ctypes.byref(down), x, t, 2, 256, P,
                                             P, 2, 2, y, t, 256, P, 1 << 30, None, None))
    refused(lib, lib.mtc_fp8_quantize(P + off, t, 2, 100, 100, P, 112, P, 2, None))
    refused(lib, lib.mtc_route_experts(P + off, t, 2, 8, 8, 2, 0, None, 1, 1, 1, 1.0, P, P, None))


@pytest.mark.parametrize("off", [1, 2])
def test_words(lib, off):
    refused(lib, lib.mtc_fp8_gemm(ctypes.byref(matrix(scales=P + off)), P, 0, 1, 256, P, 0, 128, None, 0, None, None, None))
    refused(lib, lib.mtc_fp8_matrix_init(ctypes.byref(matrix(scales=P + off))))
    refused(lib, lib.mtc_fp8_gemm(ctypes.byref(matrix()), P, 0, 1, 256, P, 0, 128, None, 0, P + off, None, None))
    refused(lib, lib.mtc_fp8_quantize(P, 0, 2, 100, 100, P, 112, P + off, 2, None))
    refused(lib, lib.mtc_fp8_pack(P + off, 4, 4, 4, P, 16, P, None))
    refused(lib, lib.mtc_fp8_pack(P, 4, 4, 4, P, 16, P + off, None))
    refused(lib, lib.mtc_fp8_unpack(ctypes.byref(matrix()), 0, P + off, 128, None))
    for bias, ids, weights in ((P + off, P, P), (None, P + off, P), (None, P, P + off)):
        refused(lib, lib.mtc_route_experts(P, 0, 2, 8, 8, 2, 0, bias, 1, 1, 1, 1.0, ids, weights, None))
    gate, down = matrix(E=4, K=256, N=128), matrix(E=4, K=128, N=256, ldk=128)
    for ids, weights, status in ((P + off, P, None), (P, P + off, None), (P, P, P + off)):
        refused(lib, lib.mtc_experts_forward(ctypes.byref(gate), ctypes.byref(gate), ctypes.byref(down), P, 0, 2, 256, ids,
                                             weights, 2, 2, P, 0, 256, P, 1 << 30, status, None))
