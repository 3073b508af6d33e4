"""The norm and gate quantisers where the forms for many and for long rows meet the other things a call may ask for."""
import os
import sys

import numpy as np
import pytest

import ternixengine_b200 as tb

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import layer_ops_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu
F = np.float32


def make(shape, dtype, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.rand(shape[0], 1, generator=g, device="cuda") * 8 + 0.01
    return (torch.randn(shape, generator=g, device="cuda") * rows).to(getattr(torch, dtype))


def check(codes, scale, t, ms, eps):
    """As the restatement: codes bit for bit, scales within the bound of an fp32 sum."""
    q, m = oracle.quantize(t)
    assert np.array_equal(codes.cpu().numpy(), q)
    want, got = oracle.row_scale64(m, ms, eps), scale.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(got[ok] - want[ok]) <= want[ok] * oracle.row_scale_bound(t.shape[1]) + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype,M,K", [("bfloat16", 3001, 2568), ("bfloat16", 450, 8192), ("float16", 450, 20480), ("float32", 3001, 1300),
                                       ("float32", 450, 10000)])
def test_many_rows_in_place_on_x(dtype, M, K):
    """The next row is on its way while this one's stream replaces x (or the residual) in memory; twice in a row, so that the
    second call's input is what the first one wrote."""
    x, r, w = make((M, K), dtype, 1), make((M, K), dtype, 2), make((1, K), dtype, 3)[0]
    for target in (x, r, x):
        h = (x.float() + r.float()).to(x.dtype)
        codes, scale, got = tb.rmsnorm_quantize(x, w, residual=r, residual_out=target)
        assert got is target and bool((target == h).all())
        hf = h.float().cpu().numpy()
        check(codes, scale, (hf * w.float().cpu().numpy()).astype(F), (hf.astype(np.float64) ** 2).mean(axis=1), 1e-5)


@pytest.mark.parametrize("dtype,K", [("float32", 16388), ("bfloat16", 32776), ("bfloat16", 32777)])
def test_rows_beyond_the_registers_and_more_of_them_than_sms(dtype, K):
    """Each CTA walks several rows in two passes; zero and poisoned rows between others, the stream in place."""
    M = 333
    x, r = make((M, K), dtype, 4), make((M, K), dtype, 5)
    x[7], r[7] = 0, 0
    x[150, K - 1] = float("nan")
    z = (np.where(x.float().cpu().numpy() < 0, F(0), x.float().cpu().numpy()) * r.float().cpu().numpy()).astype(F)
    check(*tb.glu_quantize(x, r, activation="relu"), z, None, None)
    hf = (x.float() + r.float()).to(x.dtype).float().cpu().numpy()
    codes, scale, h = tb.rmsnorm_quantize(x, residual=r, residual_out=x)
    assert h is x and np.array_equal(h.float().cpu().numpy(), hf, equal_nan=True)
    with np.errstate(invalid="ignore"):
        check(codes, scale, hf, (hf.astype(np.float64) ** 2).mean(axis=1), 1e-5)
