"""What the entry points around the product refuse before they touch a pointer or a GPU, and what they accept as nothing to
do; and the CPU restatement that the GPU tests compare with."""
import ctypes
import os
import sys

import numpy as np
import pytest

import ternixengine_b200 as tb

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import layer_ops_oracle as oracle  # noqa: E402

P = 1 << 20          # an address that is never dereferenced: every call below returns before a launch
NAN = float("nan")


def norm(x=P, ldx=64, r=None, ldr=0, dt=1, w=None, wdt=0, eps=1e-5, h=None, ldh=0, a=P, s=P, M=4, K=64):
    return tb.lib.ternix_b200_rmsnorm_quantize(x, ldx, r, ldr, dt, w, wdt, eps, h, ldh, a, s, M, K, None)


def glu(g=P, ldg=64, u=P, ldu=64, dt=1, act=3, norm=0, w=None, wdt=0, eps=0.0, a=P, s=P, M=4, K=64):
    return tb.lib.ternix_b200_glu_quantize(g, ldg, u, ldu, dt, act, norm, w, wdt, eps, a, s, M, K, None)


def fused(a=P, w=P, y=P, ldy=64, M=4, K=64, N=64, kernel=0, rs=P, cs=None, act=0, bias=None, bdt=0, dt=1, res=None, ldr=0, ep=True):
    e = tb._Epilogue(row_scale=rs, col_scale=cs, w_scale=1.0, activation=act, bias=bias, bias_dtype=bdt, out_dtype=dt, residual=res, ldr=ldr)
    return tb.lib.ternix_b200_matmul_fused(a, w, ctypes.byref(e) if ep else None, y, ldy, M, K, N, kernel, None, None)


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), tb.ERR_INVALID_SHAPE), (dict(K=-1), tb.ERR_INVALID_SHAPE), (dict(dt=3), tb.ERR_INVALID_ARG),
    (dict(dt=-1), tb.ERR_INVALID_ARG), (dict(x=None), tb.ERR_INVALID_ARG), (dict(a=None), tb.ERR_INVALID_ARG),
    (dict(s=None), tb.ERR_INVALID_ARG), (dict(ldx=63), tb.ERR_INVALID_ARG), (dict(eps=0.0), tb.ERR_INVALID_ARG),
    (dict(eps=NAN), tb.ERR_INVALID_ARG), (dict(eps=-1.0), tb.ERR_INVALID_ARG), (dict(eps=1.5), tb.ERR_INVALID_ARG),
    (dict(r=P, ldr=64), tb.ERR_INVALID_ARG), (dict(h=P, ldh=64), tb.ERR_INVALID_ARG),
    (dict(r=P, h=P, ldr=63, ldh=64), tb.ERR_INVALID_ARG), (dict(r=P, h=P, ldr=64, ldh=63), tb.ERR_INVALID_ARG),
    (dict(w=P, wdt=2), tb.ERR_INVALID_ARG), (dict(w=P, wdt=7), tb.ERR_INVALID_ARG), (dict(w=P + 1, wdt=1), tb.ERR_INVALID_ARG),
    (dict(x=P + 1), tb.ERR_INVALID_ARG), (dict(dt=0, x=P + 2), tb.ERR_INVALID_ARG), (dict(s=P + 2), tb.ERR_INVALID_ARG),
    (dict(M=0), tb.OK), (dict(M=0, x=None, a=None, s=None), tb.OK),
])
def test_rmsnorm_quantize_arguments(kw, code):
    assert norm(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), tb.ERR_INVALID_SHAPE), (dict(K=-1), tb.ERR_INVALID_SHAPE), (dict(dt=3), tb.ERR_INVALID_ARG),
    (dict(act=-1), tb.ERR_INVALID_ARG), (dict(act=6), tb.ERR_INVALID_ARG), (dict(g=None), tb.ERR_INVALID_ARG),
    (dict(u=None), tb.ERR_INVALID_ARG), (dict(a=None), tb.ERR_INVALID_ARG), (dict(s=None), tb.ERR_INVALID_ARG),
    (dict(ldg=63), tb.ERR_INVALID_ARG), (dict(ldu=0), tb.ERR_INVALID_ARG), (dict(norm=1, eps=0.0), tb.ERR_INVALID_ARG),
    (dict(norm=1, eps=NAN), tb.ERR_INVALID_ARG), (dict(w=P, wdt=1), tb.ERR_INVALID_ARG),
    (dict(norm=1, eps=1e-5, w=P, wdt=2), tb.ERR_INVALID_ARG), (dict(u=P + 1), tb.ERR_INVALID_ARG), (dict(M=0), tb.OK),
])
def test_glu_quantize_arguments(kw, code):
    assert glu(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), tb.ERR_INVALID_SHAPE), (dict(N=-4), tb.ERR_INVALID_SHAPE), (dict(N=66), tb.ERR_INVALID_SHAPE),
    (dict(K=-1), tb.ERR_INVALID_SHAPE), (dict(ep=False), tb.ERR_INVALID_ARG), (dict(ldy=63), tb.ERR_INVALID_ARG),
    (dict(kernel=6), tb.ERR_INVALID_ARG), (dict(kernel=-1), tb.ERR_INVALID_ARG), (dict(act=6), tb.ERR_INVALID_ARG),
    (dict(dt=3), tb.ERR_INVALID_ARG), (dict(bias=P, bdt=3), tb.ERR_INVALID_ARG), (dict(bias=P + 2), tb.ERR_INVALID_ARG),
    (dict(res=P, ldr=63), tb.ERR_INVALID_ARG), (dict(rs=None), tb.ERR_INVALID_ARG), (dict(a=None), tb.ERR_INVALID_ARG),
    (dict(w=None), tb.ERR_INVALID_ARG), (dict(y=None), tb.ERR_INVALID_ARG), (dict(y=P + 1), tb.ERR_INVALID_ARG),
    (dict(dt=0, y=P + 2), tb.ERR_INVALID_ARG), (dict(res=P + 1, ldr=64), tb.ERR_INVALID_ARG), (dict(rs=P + 1), tb.ERR_INVALID_ARG),
    (dict(cs=P + 2), tb.ERR_INVALID_ARG), (dict(kernel=tb.KERNEL_GEMV, M=17), tb.ERR_UNSUPPORTED),
    (dict(kernel=tb.KERNEL_SKINNY_TC), tb.ERR_UNSUPPORTED), (dict(kernel=tb.KERNEL_DECODE_MMA, K=65), tb.ERR_UNSUPPORTED),
    (dict(kernel=tb.KERNEL_GEMM_TC, N=68, ldy=68), tb.ERR_UNSUPPORTED), (dict(kernel=tb.KERNEL_GEMM_TC, a=P + 1), tb.ERR_UNSUPPORTED),
    (dict(M=0), tb.OK), (dict(N=0), tb.OK),
])
def test_matmul_fused_arguments(kw, code):
    assert fused(**kw) == code


def test_python_refuses_cpu_tensors():
    import torch
    x = torch.zeros(2, 64)
    for call in (lambda: tb.rmsnorm_quantize(x), lambda: tb.glu_quantize(x, x),
                 lambda: tb.matmul_fused(x.to(torch.int8), torch.zeros(64, 16, dtype=torch.uint8), torch.ones(2))):
        with pytest.raises(ValueError):
            call()


def test_restatement():
    """The restatement's own anchors: ties to even, signs, zero rows, poisoned rows, activations at known points."""
    t = np.array([[127, 0.5, 1.5, -0.5, -2.5], [0, 0, 0, 0, 0], [1, np.inf, 0, 0, 0], [1, np.nan, 0, 0, 0],
                  [2e-45, 0, -2e-45, 0, 0]], dtype=np.float32)
    q, m = oracle.quantize(t)
    assert q.tolist() == [[127, 0, 2, 0, -2], [0] * 5, [0] * 5, [0] * 5, [127, 0, -127, 0, 0]]
    s = oracle.row_scale64(m, np.array([3.0] * 5), 1.0)
    assert s[0] == 0.5 and s[1] == 1 and np.isnan(s[2]) and np.isnan(s[3])
    assert oracle.activate64(np.array([-2.0, 3.0]), "relu2").tolist() == [0, 9]
    assert abs(oracle.activate64(np.array([1.0]), "silu")[0] - 0.7310585786300049) < 1e-15
    assert abs(oracle.activate64(np.array([1.0]), "gelu")[0] - 0.8413447460685429) < 1e-15
    assert abs(oracle.activate64(np.array([1.0]), "gelu_tanh")[0] - 0.8411919906082768) < 1e-12


def test_the_short_way_leaves_the_rest():
    """The compiled way from Python to the C ABI answers None, with no error left behind, for whatever it does not take."""
    import torch
    rt = tb._rt()
    x, q, s = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    w = torch.zeros(64, 16, dtype=torch.uint8)

    class Odd:
        dtype, shape = torch.float32, (2, 64)

        def get_device(self):
            raise RuntimeError("no device")

    for call, args in [(rt.norm, ()), (rt.norm, (1,) * 7), (rt.norm, (None,) * 7), (rt.norm, (x, None, None, 1e-5, q, s, None)),
                       (rt.norm, (x, None, None, 1, q, s, None)), (rt.norm, (Odd(), None, None, 1e-5, q, s, None)),
                       (rt.norm, (x, None, x, 1e-5, q, s, None)), (rt.glu, ("x",) * 7), (rt.glu, (x, x, None, None, None, q, s)),
                       (rt.glu, (x, x, 3, s, None, q, s)), (rt.glu, (Odd(), x, 3, None, None, q, s)), (rt.glu, (x, x, 1 << 70, None, None, q, s)),
                       (rt.product, ()), (rt.product, (q, w, s, 1.0, None, 0, None, x, 0)), (rt.product, (q, w, s, 1.0, None, None, None, x, 0)),
                       (rt.product, (Odd(), w, s, 1.0, None, 0, None, x, 0)), (rt.product, (q, w, s, "1", None, 0, None, x, None))]:
        assert call(*args) is None
