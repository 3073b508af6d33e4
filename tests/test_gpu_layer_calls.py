"""The layer operators' calls as a program makes them: the short way (every output given) against the long one, malformed
operands with every output given, the same tensor twice, two host threads, and a process whose first call is captured."""
import os
import subprocess
import sys
import threading

import pytest

import ternixengine_b200 as tb

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def padded(M, K, dtype, seed, pad=8):
    """(M, K) values in rows of K + pad."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(M, K + pad, generator=g, device="cuda").to(dtype)[:, :K]


def layer(M, K, N, seed=0):
    import torch
    a = torch.from_numpy(tb.synth_activations((M, K), seed)).cuda()
    w = torch.from_numpy(tb.synth_packed_weights(K, N, seed)).cuda()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return a, w, torch.rand(M, generator=g, device="cuda") + 0.5, torch.rand(N, generator=g, device="cuda") + 0.5


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("M,K", [(1, 64), (5, 640), (3, 1001)])
def test_short_and_long_way_agree(M, K, dtype):
    import torch
    T = getattr(torch, dtype)
    x, r = padded(M, K, T, 1), padded(M, K, T, 2)
    calls = tb._rt()
    for w in (None, torch.rand(K, device="cuda"), torch.rand(K, device="cuda").to(T)):
        for res in (None, r):
            want = tb.rmsnorm_quantize(x, w, residual=res, eps=1e-6)
            out = [torch.full_like(want[0], 99), torch.full_like(want[1], 99)]
            h = None if res is None else padded(M, K, T, 3)
            assert calls.norm(x, w, res, 1e-6, out[0], out[1], h) == 0
            assert all(torch.equal(p, q) for p, q in zip(out + ([] if h is None else [h]), want))
            got = tb.rmsnorm_quantize(x, w, residual=res, eps=1e-6, out=out[0], row_scale=out[1], residual_out=h)
            assert got[0] is out[0] and got[1] is out[1] and (h is None or got[2] is h)
        eps = None if w is None else 1e-5
        for act in tb.ACTIVATIONS:
            want = tb.glu_quantize(x, r, activation=act, weight=w, eps=eps)
            out = [torch.full_like(want[0], 99), torch.full_like(want[1], 99)]
            assert calls.glu(x, r, tb.ACTIVATIONS[act], w, eps, *out) == 0
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    N = 192
    a, wp, rs, cs = layer(M, K, N)
    res = padded(M, N, T, 5)
    for scale in (0.25, cs):
        for bias in (None, cs, cs.bfloat16(), cs.half()):
            for residual in (None, res):
                want = tb.matmul_fused(a, wp, rs, scale, bias=bias, activation="silu", residual=residual, out_dtype=T)
                out = padded(M, N, T, 6)
                assert calls.product(a, wp, rs, scale, bias, tb.ACTIVATIONS["silu"], residual, out, tb.KERNELS["auto"]) == 0
                assert torch.equal(out, want)


def test_malformed_operands_with_every_output_given():
    """Nothing is launched: the call raises, and the outputs keep what they held."""
    import torch
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, s, h = torch.full((4, 64), 7, dtype=torch.int8, device="cuda"), torch.full((4,), 7.0, device="cuda"), torch.full_like(x, 7)

    def norm(x=x, weight=w, residual=x, eps=1e-5, out=q, row_scale=s, residual_out=h):
        return tb.rmsnorm_quantize(x, weight, residual=residual, eps=eps, out=out, row_scale=row_scale, residual_out=residual_out)

    def glu(gate=x, up=x, activation="silu", weight=None, eps=None, out=q, row_scale=s):
        return tb.glu_quantize(gate, up, activation=activation, weight=weight, eps=eps, out=out, row_scale=row_scale)

    a, wp, rs, cs = layer(4, 64, 64)
    y = torch.full((4, 64), 7, dtype=torch.bfloat16, device="cuda")

    def product(a=a, w=wp, row_scale=rs, w_scale=cs, out=y, **kw):
        return tb.matmul_fused(a, w, row_scale, w_scale, out=out, **kw)

    wide = torch.zeros((4, 128), dtype=torch.int8, device="cuda")
    bad = [
        lambda: norm(x=x.cpu()), lambda: norm(x=x.double()), lambda: norm(x=x.t()), lambda: norm(x=x[0]),
        lambda: norm(x=x[:1].expand(4, 64)), lambda: norm(weight=w[:63]), lambda: norm(weight=w.half()), lambda: norm(weight=w.cpu()),
        lambda: norm(weight=w[None]), lambda: norm(residual=x.float()), lambda: norm(residual=x[:3]), lambda: norm(residual=None),
        lambda: norm(eps=0.0), lambda: norm(eps=float("nan")), lambda: norm(out=wide[:, :64]), lambda: norm(out=q.cpu()),
        lambda: norm(out=q.view(torch.uint8)), lambda: norm(row_scale=s[:3]), lambda: norm(row_scale=s.double()),
        lambda: norm(row_scale=s.cpu()), lambda: norm(residual_out=h.float()), lambda: norm(residual_out=h[:1].expand(4, 64)),
        lambda: glu(gate=x.cpu()), lambda: glu(up=x.half()), lambda: glu(up=x[:, :32]), lambda: glu(activation="swish"),
        lambda: glu(weight=w), lambda: glu(weight=w[:3], eps=1e-5), lambda: glu(eps=0.0), lambda: glu(out=wide[:, :64]),
        lambda: glu(row_scale=s[:3]),
        lambda: product(a=a.cpu()), lambda: product(a=a.float()), lambda: product(a=a[:, :32]), lambda: product(a=wide[:, :64]),
        lambda: product(w=wp.cpu()), lambda: product(w=wp.view(torch.int8)), lambda: product(w=wp[:, ::2]), lambda: product(row_scale=rs[:3]),
        lambda: product(row_scale=rs.half()), lambda: product(row_scale=rs.cpu()), lambda: product(w_scale=cs[:63]), lambda: product(w_scale=cs.half()),
        lambda: product(w_scale=cs.cpu()), lambda: product(bias=cs[:3]), lambda: product(bias=cs.double()), lambda: product(bias=cs.cpu()),
        lambda: product(activation="tanh"), lambda: product(kernel="fast"),
        lambda: product(kernel="skinny_tc"),       # no fused form
        lambda: product(residual=y.float()), lambda: product(residual=y[:1].expand(4, 64)),
        lambda: product(residual=y.cpu()), lambda: product(out=y.int()), lambda: product(out=y.cpu()), lambda: product(out=y.t()),
        lambda: product(out=y[:1].expand(4, 64)), lambda: product(out_dtype=torch.float32),
        lambda: product(status=torch.zeros(1, dtype=torch.int32)), lambda: product(status=torch.zeros(1, device="cuda")),
        lambda: product(status=torch.zeros(0, dtype=torch.int32, device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")
    for call in (lambda: norm(x=None), lambda: glu(up=3), lambda: product(w="w"), lambda: product(w_scale="1")):
        with pytest.raises((AttributeError, TypeError)):
            call()
    torch.cuda.synchronize()
    assert (q == 7).all() and (s == 7).all() and (h == 7).all() and (y == 7).all()


def test_the_same_tensor_twice():
    """x + x in place, a gate that is its own partner, a product onto its own output, one weight matrix in two calls."""
    import torch
    x = padded(9, 640, torch.bfloat16, 1, pad=0)
    want = tb.rmsnorm_quantize(x.clone(), residual=x.clone())
    y = x.clone()
    got = tb.rmsnorm_quantize(y, residual=y, residual_out=y)
    assert got[2] is y and all(torch.equal(p, q) for p, q in zip(got, want))
    assert all(torch.equal(p, q) for p, q in zip(tb.glu_quantize(x, x, activation="relu"), tb.glu_quantize(x, x.clone(), activation="relu")))
    a, w, rs, cs = layer(9, 640, 640)
    r = x.clone()
    want = tb.matmul_fused(a, w, rs, cs, bias=cs, residual=r.clone())
    assert tb.matmul_fused(a, w, rs, cs, bias=cs, residual=r, out=r) is r and torch.equal(r, want)


def test_status_word():
    import torch
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for M in (1, 4, 40, 300):
        a, w, rs, cs = layer(M, 640, 640)
        y = tb.matmul_fused(a, w, rs, cs, status=status)
        assert torch.equal(y, tb.matmul_fused(a, w, rs, cs)) and int(status) == 0


def test_two_host_threads():
    """Each on a stream of its own, with products that share the library's scratch pool among the calls."""
    import torch
    sizes = [(3, 640, 640), (40, 1024, 640), (33, 1029, 1028)]
    ops = [layer(*s, seed=i) for i, s in enumerate(sizes)]
    xs = [padded(s[0], 640, torch.bfloat16, i) for i, s in enumerate(sizes)]

    def once(i):
        a, w, rs, cs = ops[i]
        return [tb.matmul_fused(a, w, rs, cs, activation="silu"), *tb.rmsnorm_quantize(xs[i]), *tb.glu_quantize(xs[i], xs[i])]

    want = [once(i) for i in range(len(sizes))]
    torch.cuda.synchronize()
    bad = []

    def work(turn):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for rep in range(30):
                    i = (rep + turn) % len(sizes)
                    got = once(i)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                        bad.append((turn, rep, i))
        except Exception as e:             # a thread's own exception would not reach the test
            bad.append(e)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


FIRST_CALL_CAPTURED = """
import torch, ternixengine_b200 as tb
M, K, N = {sizes}
x = torch.randn(M, K, device="cuda").bfloat16()
w = torch.from_numpy(tb.synth_packed_weights(K, N, 1)).cuda()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q, s = tb.rmsnorm_quantize(x)
    y = tb.matmul_fused(q, w, s, 0.05)
    q2, s2 = tb.glu_quantize(y, y, activation="relu2")
for _ in range(2):
    x.copy_(torch.randn(M, K, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    q_, s_ = tb.rmsnorm_quantize(x)
    y_ = tb.matmul_fused(q_, w, s_, 0.05)
    for p, r in zip((q, s, y, q2, s2), (q_, s_, y_, *tb.glu_quantize(y_, y_, activation="relu2"))):
        assert torch.equal(p, r)
print("replayed")
"""


@pytest.mark.parametrize("sizes", [(1, 2560, 640), (6, 2560, 640), (40, 2560, 640), (300, 1040, 832), (33, 1029, 1028), (3, 65, 68)])
def test_first_call_of_a_process_is_captured(sizes):
    """Everything that the library sets up on first use (attributes, occupancy, its pool) may happen under capture."""
    env = dict(os.environ, PYTHONPATH=ROOT)
    p = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED.format(sizes=sizes)], capture_output=True, text=True, timeout=300, env=env)
    assert p.returncode == 0 and "replayed" in p.stdout, p.stderr[-2000:]
