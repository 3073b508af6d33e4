"""CPU restatement of the steps around the ternary product in a quantised layer -- TEST INFRASTRUCTURE ONLY.

Parity unpinned, as for bitnet_scaling_oracle.py: the reference has an fp32 RMSNorm and a SwiGLU over interleaved pairs
(src/simd_math.cpp:7-46) but neither joined with a residual or a quantiser.  Two forms of each step:
  * in float32 with the operation order written out, where every operation is exactly rounded on both sides (sums, products,
    quotients, comparisons), so that codes and outputs can be compared bit for bit;
  * in float64 from the formula, with the bound that the fp32 arithmetic of the kernels has to keep.
"""
import math

import numpy as np

F = np.float32
_ERFC = np.vectorize(math.erfc, otypes=[np.float64])


def activate64(v, act):
    """The activation in float64."""
    v = np.asarray(v, dtype=np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if act == "relu":
            return np.where(v < 0, 0.0, v)
        if act == "relu2":
            return np.where(v < 0, 0.0, v) ** 2
        if act == "silu":
            return v / (1 + np.exp(-v))
        if act == "gelu":
            return v * _ERFC(-v / math.sqrt(2)) / 2                 # 1 + erf(x) = erfc(-x), without the cancellation
        if act == "gelu_tanh":
            # (1 + tanh u) / 2 = 1 / (1 + exp(-2u)), without the cancellation
            return v / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def activation_error(v, act):
    """Absolute error that an fp32 evaluation of the activation may have, beside one rounding of its result.

    relu and relu2 are exactly rounded.  silu = v / (1 + e), e = exp(-v) from the hardware's exponential: its documented
    error is 2 + 1.173 |v| units in the last place (2^-23), the sum rounds once (2^-24) and the quotient has 2 ulp, so the
    result is off by at most its own size x (2 + 1.173 |v| + 3) x 2^-23.  gelu_tanh is the same with the argument 2u, which
    itself carries four roundings (4 |2u| 2^-24 in the exponent).  Both divide with the instruction that delivers 0 for
    denominators above 2^126 (documented), where the quotient is at most |v| 2^-126.  gelu = 0.5 v (1 + erf): erff has 2 ulp and its argument
    one rounding and a rounded constant (|d erf| <= 1.13 |x| 2^-23 <= 2^-23 where erf still moves), the sum one rounding of
    a value up to 2: in all |v| (2 x 2^-24 + 2^-23 + 2 x 2^-24) / 2, and two roundings of the products.  The same bound holds for
    gelu = v / (1 + 2^-w), w the base-2 logit of the normal distribution P from a fit that is off by at most 1.2e-8 in v P(v) and
    3e-8 in P: P is off by that, by P (1 - P) <= 1/4 times the exponential's 2^-22 and three roundings of w (P (1 - P) |w| <= 0.23
    in natural units, so 0.23 x 3 x 2^-24), and by 2^-22 P from sum, reciprocal and product: 1.3e-7 + 2.4e-7 P against 1.8e-7 +
    1.2e-7 P here and the 2^-24 P that every comparison adds for the result's rounding; where P nears 1 the first term vanishes
    with 1 - P.  (float32 data have smaller errors than these.)"""
    v = np.asarray(v, dtype=np.float64)
    out = np.abs(activate64(v, act))
    if act == "silu":
        return out * (5 + 1.173 * np.abs(v)) * 2.0 ** -23 + np.abs(v) * 2.0 ** -126
    if act == "gelu_tanh":
        u2 = 2 * math.sqrt(2 / math.pi) * np.abs(v + 0.044715 * v ** 3)
        return out * (5 + 3.173 * u2) * 2.0 ** -23 + np.abs(v) * 2.0 ** -126
    if act == "gelu":
        return np.abs(v) * 2.0 ** -23 * 1.5 + out * 2.0 ** -23
    return np.zeros_like(v)


def quantize(t):
    """t float32 (M, K) -> (codes int8, max|t| float32): m = max|t|, q = rint(t * (127 / m)); rows of zeros and rows with an
    infinity or NaN have codes 0.  Rows of tiny m are scaled by 2^100 first (exact)."""
    t = np.asarray(t, dtype=F)
    m = np.abs(t).max(axis=1) if t.shape[1] else np.zeros(t.shape[0], dtype=F)
    fine = np.isfinite(m) & (m > 0)
    lift = np.where(m < F(1e-30), F(2.0 ** 100), F(1))
    with np.errstate(all="ignore"):
        inv = np.where(fine, F(127) / (m * lift), F(0)).astype(F)
        v = ((t * lift[:, None]).astype(F) * inv[:, None]).astype(F)
    q = np.where(fine[:, None], np.rint(v), 0).astype(np.int8)
    return q, m


def row_scale64(m, ms, eps):
    """(m / 127) / sqrt(ms + eps) in float64; 1 for rows of zeros, NaN for rows that are not finite.  eps None: no norm."""
    m = np.asarray(m, dtype=np.float64)
    with np.errstate(all="ignore"):
        s = m / 127 if eps is None else m / 127 / np.sqrt(ms + float(F(eps)))
    s = np.where(m == 0, 1.0, s)
    return np.where(np.isfinite(m), s, np.nan)


def row_scale_bound(K):
    """Relative error of a row's scale: a sum of squares in fp32 (all terms positive: one 2^-24 for each addition on the
    longest chain, at most K / 1024 + 32 in a thread and 10 between threads, and one for the square), halved by the root, and
    six further roundings."""
    return ((K / 1024 + 32 + 10 + 1) / 2 + 6) * 2.0 ** -24
