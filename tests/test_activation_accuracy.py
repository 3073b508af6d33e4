"""How far the activations of float32 data are from their definitions, and the fit behind GELU."""
import math
import os
import re

import numpy as np
import pytest

import ternixengine_b200 as tb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = np.float32
_ERFC = np.vectorize(math.erfc, otypes=[np.float64])
FIT = 1.2e-8                       # what the fit may be off by in v P(v), as the kernels' comment states


def below(v):
    """P(-|v|), the normal distribution's smaller half."""
    return _ERFC(np.abs(v) / math.sqrt(2)) / 2


def test_the_fit_keeps_the_stated_error():
    """The kernels' coefficients, evaluated exactly: |v| times the error of P(-|v|), inside the fit's interval and beyond."""
    body = open(os.path.join(ROOT, "ternixengine_b200", "csrc", "epilogue.cuh")).read()
    body = body[body.index("float gelu_logit(float v)"):]
    body = body[:body.index("\n}")]
    top = float(re.search(r"fminf\(__fmul_rn\(v, v\), ([0-9.]+)f\)", body).group(1))
    c = [float(F(x)) for x in re.findall(r"(?:= |u, )(-?[0-9.]+(?:e-?[0-9]+)?)f", body)]
    assert len(c) == 10
    v = np.concatenate([np.linspace(0, 9, 90001), [math.sqrt(top), 12.0, 30.0]])
    u, r = np.minimum(v * v, top), np.zeros_like(v)
    for x in c:
        r = r * u + x
    e = 2.0 ** (-v * r)
    q = e / (1 + e)
    assert (v * np.abs(q - below(v))).max() <= FIT
    assert (np.diff(q[:90001]) < 0).all()                     # falls all the way, across the end of the interval too


def points(n):
    rng = np.random.default_rng(3)
    v = np.concatenate([np.linspace(-9, 9, n // 2), rng.normal(size=n // 4) * 2, rng.uniform(-90, 30, n - n // 2 - n // 4)])
    return v.astype(F)


# What follows holds for exponentials off by at most 2^-22, reciprocals by 2^-23 (their documented errors) and exact roundings.  e is
# the exponential (its argument's rounding is put back but for 2^-25 of ln 2, and rounds once: 2^-24 and 3e-9 of the argument),
# 1 + e and e / (1 + e) round once each, so q = e / (1 + e) is off by at most (4 + 1 + 1 + 2 + 1) x 2^-24 of itself.  The last
# operation is one rounding of the result.
PARTS = 9 * 2.0 ** -24


def bound(v, act):
    if act == "silu":
        q = 1 / (1 + np.exp(np.abs(v)))
        want = v / (1 + np.exp(-v))
        err = np.abs(v) * q * (PARTS + 3e-9 * np.abs(v))
    elif act == "gelu_tanh":
        w = 2 * math.sqrt(2 / math.pi) * np.abs(v + 0.044715 * v ** 3)
        q = 1 / (1 + np.exp(np.minimum(w, 700)))
        want = v / (1 + np.exp(np.clip(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3), -700, 700)))
        # the argument: two rounded constants (0.044715 and 2 sqrt(2 / pi)) and four roundings
        err = np.abs(v) * q * (PARTS + (3e-9 + 6 * 2.0 ** -24) * w)
    else:
        q = below(v)
        want = np.where(v < 0, v * q, v - v * q)
        # the logit's argument w = |v| r(v^2): rounds as the product; r by 2^-24 of the sum over its steps of u^k |partial sum|, and
        # with the rounding of u by another 2^-24 (r - r(0)).  Up to |v| = 4 all that is at most 3 x 2^-24 w; beyond, the sum is at
        # most 93 (its value at the end of the interval), so w is off by |v| (93 + 10) x 2^-24 at most, |v| <= 5.7.
        w = np.log2((1 - q) / np.maximum(q, 1e-300))
        dw = np.where(np.abs(v) <= 4, 3 * 2.0 ** -24 * w, 5.7 * 103 * 2.0 ** -24)
        err = FIT + np.abs(v) * q * (PARTS + math.log(2) * dw)
    # flushed to zero: exponentials below 2^-126, and results that are subnormal
    return want, err + np.abs(want) * 2.0 ** -24 + np.abs(v) * 2.0 ** -126 + np.finfo(F).smallest_normal


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 1 << 16), (24, 1 << 15), (300, 1 << 13)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_float32_outputs(act, M, N):
    """Through the bias of a product of zeros, in the kernel of each regime."""
    import torch
    v = points(N)
    a, w = torch.zeros(M, 64, dtype=torch.int8, device="cuda"), torch.zeros(64, N // 4, dtype=torch.uint8, device="cuda")
    y = tb.matmul_fused(a, w, torch.ones(M, device="cuda"), 1.0, bias=torch.from_numpy(v).cuda(), activation=act, out_dtype=torch.float32)
    assert torch.equal(y, y[:1].expand_as(y))
    want, tol = bound(v.astype(np.float64), act)
    off = np.abs(y[0].cpu().numpy().astype(np.float64) - want) - tol
    i = int(np.argmax(off))
    assert off[i] <= 0, (act, v[i], float(y[0, i]), want[i], tol[i])


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 5])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_float32_gates(act, K):
    """Rows of one gate value: code 127, and a scale that is |act(g)| / 127 within the same bound and the scale's own roundings (m / 127,
    and the product of m with a partner of one: exact)."""
    import torch
    v = points(4096)
    v = v[np.abs(v) > 1e-3]
    g = torch.from_numpy(v).cuda()[:, None].expand(-1, K).contiguous()
    codes, scale = tb.glu_quantize(g, torch.ones_like(g), activation=act)
    want, tol = bound(v.astype(np.float64), act)
    got = scale.cpu().numpy().astype(np.float64) * 127
    live = np.abs(want) > tol                                       # a row that may have been flushed to zeros has scale 1
    assert (np.abs(got - np.abs(want)) <= tol + np.abs(want) * 2.0 ** -23 + 127 * 2.0 ** -149)[live].all()
    assert (codes.cpu().numpy() == np.where(want < 0, -127, 127)[:, None])[live].all()
