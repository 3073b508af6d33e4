"""The longest row that the layer operators take."""
import numpy as np
import pytest

import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu


def test_longest_row():
    """2^31 - 1025 columns (4.3 GB of bfloat16): every index of the row, and the step that ends its loops, in a C int."""
    import torch
    K = 2 ** 31 - 1025
    x = torch.zeros((1, K), dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 1023, 2 ** 30, K - 1025, K - 2, K - 1]
    x[0, at] = torch.tensor([1, -2, 3, 127, -4, 5, -127], dtype=torch.bfloat16, device="cuda")
    codes, scale = tb.rmsnorm_quantize(x, eps=1e-5)
    assert codes[0, at].tolist() == [1, -2, 3, 127, -4, 5, -127] and int(torch.count_nonzero(codes)) == len(at)
    ms = (1 + 4 + 9 + 127 ** 2 + 16 + 25 + 127 ** 2) / K
    # every partial sum is a whole number below 2^24, so the sum is exact: division, addition, root, reciprocal and product round once each, and 127 / 127
    assert abs(float(scale) - 1 / np.sqrt(ms + float(np.float32(1e-5)))) <= 6 * 2.0 ** -24 * float(scale)


def test_most_rows_of_the_mma_sync_kernel():
    import torch
    M, K, N = 65536, 64, 128
    a = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda")
    w = torch.from_numpy(tb.synth_packed_weights(K, N, 1)).cuda()
    rs = torch.rand(M, device="cuda")
    assert torch.equal(tb.matmul(a, w, kernel="decode_mma"), tb.matmul(a, w, kernel="generic"))
    assert torch.equal(tb.matmul_fused(a, w, rs, 0.5, kernel="decode_mma"), tb.matmul_fused(a, w, rs, 0.5, kernel="generic"))


@pytest.mark.parametrize("K", [0, 3])
def test_more_rows_than_65535_tiles_of_the_generic_kernel(K):
    """K = 0 (nothing but the epilogue is left) and a forced kernel, at rows beyond 65535 x 32."""
    import torch
    M, N = 65535 * 32 + 37, 132
    a = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda")
    wp = tb.synth_packed_weights(K, N, 1) if K else np.zeros((0, N // 4), dtype=np.uint8)
    w = torch.from_numpy(tb.unpack_ternary(wp)).cuda().float()
    rs, bias = torch.full((M,), 0.5, device="cuda"), torch.arange(N, device="cuda").float()
    y = tb.matmul_fused(a, torch.from_numpy(wp).cuda(), rs, 1.0, bias=bias, out_dtype=torch.float32, kernel="auto" if K == 0 else "generic")
    for rows in (slice(0, 70), slice(65535 * 32 - 40, M)):
        assert torch.equal(y[rows], (a[rows].float() @ w) * 0.5 + bias)           # halves of small whole numbers: exact


def test_sizes_of_more_than_32_bits():
    """2^32 + 5 rows and 2^32 + 64 columns, which would arrive in a C int as 5 and 64."""
    import torch
    x = torch.empty((2 ** 32 + 5, 1), dtype=torch.bfloat16, device="cuda")
    w = torch.empty((1, 2 ** 30 + 16), dtype=torch.uint8, device="cuda")
    a, s = torch.ones((1, 1), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda")
    for call in (lambda: tb.rmsnorm_quantize(x), lambda: tb.rmsnorm_quantize(x.view(1, -1)), lambda: tb.glu_quantize(x, x), lambda: tb.quantize_rows(x),
                 lambda: tb.matmul_fused(a, w, s), lambda: tb.matmul(a, w), lambda: tb.matmul_dequant(a, w, s, 1.0), lambda: tb.TernaryWeights(w)):
        with pytest.raises(ValueError):
            call()
