"""Sizes at the end of a C int: what the entry points refuse before anything is launched (index arithmetic of the kernels is in
int, so a loop over 2^31 - 1 columns would pass its own end and read in front of the row)."""
import ctypes
import os
import re

import pytest

import ternixengine_b200 as tb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


class Stand:
    """What the entry points ask of a tensor, at sizes that need no memory behind them."""

    def __init__(self, dtype, *shape):
        import torch
        self.dtype, self.shape, self.is_cuda, self.device = dtype, torch.Size(shape), True, torch.device("cuda:0")

    def get_device(self):
        return 0

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def stride(self, i=None):
        strides = [1]
        for n in self.shape[:0:-1]:
            strides.insert(0, strides[0] * n)
        return tuple(strides) if i is None else strides[i]

    def data_ptr(self):
        raise AssertionError("asked for an address before the sizes were checked")


BEYOND = [MAX + 1, 2 ** 32 + 8]      # the second would arrive in a C int as 8


@pytest.mark.parametrize("n", BEYOND)
def test_python_refuses_before_it_hands_sizes_on(n):
    import torch
    bf16, f32, i8, u8 = torch.bfloat16, torch.float32, torch.int8, torch.uint8
    for shape in ((n, 1), (1, n)):
        x, q, s = Stand(bf16, *shape), Stand(i8, *shape), Stand(f32, shape[0])
        for call in (lambda: tb.rmsnorm_quantize(x), lambda: tb.rmsnorm_quantize(x, residual=x, out=q, row_scale=s, residual_out=x),
                     lambda: tb.glu_quantize(x, x), lambda: tb.glu_quantize(x, x, out=q, row_scale=s), lambda: tb.quantize_rows(x)):
            with pytest.raises(ValueError, match="sizes go up to"):
                call()
    for M, K, N in ((n, 1, 4), (1, n, 4), (1, 1, n // 4 * 4 + 4)):
        a, w, s = Stand(i8, M, K), Stand(u8, K, N // 4), Stand(f32, M)
        for call in (lambda: tb.matmul_fused(a, w, s), lambda: tb.matmul_fused(a, w, s, out=Stand(bf16, M, N)), lambda: tb.matmul(a, w),
                     lambda: tb.matmul_dequant(a, w, s, 1.0), lambda: tb.ProjectionGroup([(a, w, Stand(torch.int32, M, N))])):
            with pytest.raises(ValueError, match="sizes go up to"):
                call()
    with pytest.raises(ValueError, match="sizes go up to"):
        tb.TernaryWeights(Stand(u8, n, 1))
    with pytest.raises(ValueError, match="sizes go up to"):
        tb.prepack_k4(Stand(u8, n, 1))


def test_the_limit_is_the_headers():
    header = open(os.path.join(ROOT, "include", "ternix_b200.h")).read()
    assert int(re.search(r"TERNIX_B200_MAX_SIZE (\d+)", header).group(1)) == tb.MAX_SIZE == MAX
