"""Sizes at the end of a C int: what the entry points refuse before anything is launched (index arithmetic of the kernels is in
int, so a loop over 2^31 - 1 columns would pass its own end and read in front of the row)."""
import ctypes

import pytest

import ternixengine_b200 as tb

P = 1 << 20          # an address that is never dereferenced: every call below returns before a launch
MAX = 2 ** 31 - 1025
TOO_LARGE = [MAX + 1, 2 ** 31 - 1]


@pytest.mark.parametrize("n", TOO_LARGE)
def test_layer_operators(n):
    norm, glu, fused = tb.lib.ternix_b200_rmsnorm_quantize, tb.lib.ternix_b200_glu_quantize, tb.lib.ternix_b200_matmul_fused
    for M, K in ((1, n), (n, 1)):
        assert norm(P, K, None, 0, 1, None, 0, 1e-5, None, 0, P, P, M, K, None) == tb.ERR_INVALID_SHAPE
        assert norm(P, K, P, K, 0, P, 0, 1e-5, P, K, P, P, M, K, None) == tb.ERR_INVALID_SHAPE
        assert glu(P, K, P, K, 1, 3, 0, None, 0, 0.0, P, P, M, K, None) == tb.ERR_INVALID_SHAPE
    ep = tb._Epilogue(row_scale=P, w_scale=1.0, out_dtype=1)
    for M, K, N in ((1, n, 4), (n, 1, 4), (1, 1, n // 4 * 4)):
        if max(M, K, N) > MAX:
            assert fused(P, P, ctypes.byref(ep), P, N, M, K, N, 0, None, None) == tb.ERR_INVALID_SHAPE


@pytest.mark.parametrize("n", TOO_LARGE)
def test_products(n):
    for M, K, N in ((1, n, 4), (n, 1, 4), (1, 1, n // 4 * 4)):
        if max(M, K, N) <= MAX:
            continue
        assert tb.lib.ternix_b200_matmul_ex(P, P, P, M, K, N, N, 0, None, None) == tb.ERR_INVALID_SHAPE
        assert tb.lib.ternix_b200_matmul(P, P, P, M, K, N, None) == tb.ERR_INVALID_SHAPE
        dest = (ctypes.c_void_p * 1)(P)
        assert tb.lib.ternix_b200_matmul_dequant(P, P, dest, 1, P, 1.0, M, K, N, N, None, None) == tb.ERR_INVALID_SHAPE
    assert tb.lib.ternix_b200_quantize_rows(P, 0, n, P, P, 1, n, None) == tb.ERR_INVALID_SHAPE


def test_nothing_to_do_stays_nothing():
    assert tb.lib.ternix_b200_rmsnorm_quantize(None, MAX, None, 0, 1, None, 0, 1e-5, None, 0, None, None, 0, MAX, None) == tb.OK
    assert tb.lib.ternix_b200_matmul_ex(None, None, None, 0, MAX, 4, 4, 0, None, None) == tb.OK


def test_rows_of_the_mma_sync_kernel():
    """Its work items hold a row in 16 bits: row 65536 would be row 0 again."""
    ep = tb._Epilogue(row_scale=P, w_scale=1.0, out_dtype=1)
    for M in (65537, 70000):
        assert tb.lib.ternix_b200_matmul_fused(P, P, ctypes.byref(ep), P, 64, M, 64, 64, tb.KERNEL_DECODE_MMA, None, None) == tb.ERR_UNSUPPORTED
        assert tb.lib.ternix_b200_matmul_ex(P, P, P, M, 64, 64, 64, tb.KERNEL_DECODE_MMA, None, None) == tb.ERR_UNSUPPORTED
