"""Rows taken as single elements: what is chosen by type, length and number of rows, next to its neighbours in size."""
import pytest

import ternixengine_b200 as tb
from test_gpu_row_quant_more import F, check, make

import numpy as np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,M,K", [("float32", m, k) for m in (2, 400) for k in (3, 4096, 4097, 8192, 8193, 16383, 16384, 16385)] +
                         [(d, m, k) for d in ("bfloat16", "float16") for m, k in ((2, 639), (1300, 641), (400, 1023), (1300, 1023), (5, 1025))])
def test_rows_at_any_offset(dtype, M, K):
    """Operands at offsets and pitches of their own, nothing outside the rows read or written; the stream in place; a zero row and a
    poisoned one."""
    import torch

    def at(offset, pitch, values, fill):
        flat = torch.full((offset + M * pitch + 16,), fill, dtype=values.dtype, device="cuda")
        view = flat[offset:offset + M * pitch].view(M, pitch)[:, :K]
        view.copy_(values)
        return flat, view

    x0, r0, w = make((M, K), dtype, 1), make((M, K), dtype, 2), make((1, K), dtype, 3)[0]
    x0[0], r0[0] = 0, 0
    x0[M - 1, K // 2] = float("nan")
    _, x = at(1, K + 3, x0, float("inf"))
    r_flat, r = at(2, K + 5, r0, float("inf"))
    xf, rf, wf = x0.float().cpu().numpy(), r0.float().cpu().numpy(), w.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        z = (np.where(xf < 0, F(0), xf) * rf).astype(F)
        check(*tb.glu_quantize(x, r, activation="relu", weight=w, eps=1e-5), (z * wf).astype(F), (z.astype(np.float64) ** 2).mean(axis=1), 1e-5)
        check(*tb.glu_quantize(x, r, activation="relu"), z, None, None)
        hf = (x0.float() + r0.float()).to(x0.dtype).float().cpu().numpy()
        codes, scale, h = tb.rmsnorm_quantize(x, w, residual=r, residual_out=r)
        assert h is r and np.array_equal(r.float().cpu().numpy(), hf, equal_nan=True)
        check(codes, scale, (hf * wf).astype(F), (hf.astype(np.float64) ** 2).mean(axis=1), 1e-5)
        check(*tb.rmsnorm_quantize(x, w), (xf * wf).astype(F), (xf.astype(np.float64) ** 2).mean(axis=1), 1e-5)
    r.fill_(float("inf"))
    assert bool((r_flat == float("inf")).all())
