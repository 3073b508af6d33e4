"""The product with scales, bias, activation and residual in its epilogue (matmul_fused) on the GPU.  The integer product
comes from the CPU oracle; what follows it is restated in float32, operation by operation, and compared bit for bit where
every operation is exactly rounded (no activation, relu, relu2), within the activation's error otherwise."""
import os
import sys

import numpy as np
import pytest

import oracle_lib
import ternixengine_b200 as tb

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import layer_ops_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu

F = np.float32
# one row; row groups of 8 and 16, clusters along K and not; 64- and 128-row tensor-memory decode; prefill tiles, whole
# and ragged in both directions; narrow outputs
ALIGNED = [(1, 64, 64), (1, 2560, 6912), (1, 16, 128), (2, 2560, 640), (3, 1040, 320), (8, 128, 4160), (16, 4096, 1024),
           (17, 272, 576), (32, 4096, 1088), (33, 8192, 128), (48, 1024, 2112), (64, 2560, 704), (65, 272, 576),
           (100, 4096, 1024), (128, 2560, 640), (129, 272, 1984), (200, 256, 64), (300, 1040, 832), (513, 2560, 1344)]
# sizes that no aligned copy fits: small ones as they are, large ones through an aligned copy
RAGGED = [(1, 1, 4), (1, 129, 4), (7, 129, 132), (31, 1029, 2052), (1, 3001, 1028), (5, 1024, 100), (33, 100, 64),
          (16, 1001, 320), (255, 2561, 1732), (129, 1029, 2052), (20, 4099, 4100), (40, 3001, 2052), (300, 1030, 2112),
          (1, 20001, 12004), (300, 2560, 1028)]
ACTS = list(tb.ACTIVATIONS)


def operands(M, K, N, seed):
    import torch
    a = tb.synth_activations((M, K), seed)
    wp = tb.synth_packed_weights(K, N, seed + 1)
    rng = np.random.default_rng(seed)
    rs = rng.uniform(1e-3, 0.05, size=M).astype(F)
    cs = rng.uniform(1e-3, 0.05, size=N).astype(F)
    return a, wp, rs, cs, torch.from_numpy(a).cuda(), torch.from_numpy(wp).cuda(), torch.from_numpy(rs).cuda(), torch.from_numpy(cs).cuda()


def check(y, c, rs, cs, bias, act, residual):
    """y against the restatement on the exact product c; bias and residual are float32 arrays of what the kernel reads."""
    import torch
    v = ((c.astype(F) * rs[:, None]).astype(F) * cs).astype(F)
    if bias is not None:
        v = (v + bias[None, :]).astype(F)
    if act in ("none", "relu", "relu2"):
        w = v if act == "none" else np.where(v < 0, F(0), v)
        w = (w * w).astype(F) if act == "relu2" else w
        if residual is not None:
            w = (w + residual).astype(F)
        want = torch.from_numpy(w).to(y.dtype)
        assert torch.equal(y.cpu() + 0.0, want + 0.0)          # + 0.0: a zero's sign is not part of the contract
        return
    want = oracle.activate64(v, act)
    tol = oracle.activation_error(v, act) + np.abs(want) * 2.0 ** -24
    if residual is not None:
        want = want + residual.astype(np.float64)
        tol = tol + np.abs(want) * 2.0 ** -24
    tol = tol + (np.abs(want) + tol) * torch.finfo(y.dtype).eps / 2 + torch.finfo(y.dtype).smallest_normal
    got = y.double().cpu().numpy()
    off = np.abs(got - want) - tol
    at = np.unravel_index(np.argmax(off), off.shape)
    assert off[at] <= 0, (at, act, v[at], got[at], want[at], tol[at])


@pytest.mark.parametrize("shape", ALIGNED + RAGGED)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_every_regime(shape, dtype):
    import torch
    M, K, N = shape
    t = getattr(torch, dtype)
    a, wp, rs, cs, ta, tw, trs, tcs = operands(M, K, N, M + K + N)
    c = oracle_lib.matmul(a, wp)
    g = torch.Generator(device="cuda").manual_seed(M)
    bias = torch.randn(N, generator=g, device="cuda")
    residual = (torch.randn(M, N, generator=g, device="cuda") * 3).to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = tb.matmul_fused(ta, tw, trs, 0.0371, out_dtype=t, status=status)
    check(y, c, rs, F(0.0371), None, "none", None)
    for i, act in enumerate(ACTS):
        b = None if i == 0 else bias if i % 2 else bias.to(torch.bfloat16 if i == 2 else torch.float16)
        r = residual if i in (0, 2, 3) else None
        y = tb.matmul_fused(ta, tw, trs, tcs if i != 4 else 0.02, bias=b, activation=act, residual=r, out_dtype=t, status=status)
        check(y, c, rs, cs[None, :] if i != 4 else F(0.02), None if b is None else b.float().cpu().numpy(), act,
              None if r is None else r.float().cpu().numpy())
    assert int(status.item()) == 0


@pytest.mark.parametrize("shape", [(1, 2560, 640), (9, 1040, 576), (40, 1024, 832), (100, 2560, 640), (300, 1040, 832)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("act", ACTS)
def test_kernels_give_the_same_bits(shape, dtype, act):
    """Every kernel that takes the problem, at output pitches that allow vector accesses and that do not."""
    import torch
    M, K, N = shape
    t = getattr(torch, dtype)
    _, _, _, _, ta, tw, trs, tcs = operands(M, K, N, 3)
    bias = torch.randn(N, device="cuda").half()
    wide_r = torch.randn(M, N + 7, device="cuda").to(t)
    want = None
    for kernel in ("auto", "generic", "gemv", "decode_mma", "skinny_tc", "gemm_tc"):
        if kernel == "gemv" and M > 16 or kernel == "skinny_tc":           # the latter has no fused form
            with pytest.raises(ValueError):
                tb.matmul_fused(ta, tw, trs, tcs, kernel=kernel)
            continue
        for pad in (0, 5, 16):
            wide = torch.full((M + 1, N + pad), 9.0, dtype=t, device="cuda")
            y = tb.matmul_fused(ta, tw, trs, tcs, bias=bias, activation=act, residual=wide_r[:, 1:N + 1] if pad == 5 else wide_r[:, 1:N + 1].contiguous(),
                                out=wide[:M, pad // 2:pad // 2 + N], kernel=kernel)
            want = y.clone() if want is None else want
            assert torch.equal(y, want), (kernel, pad)
            y.fill_(9.0)
            assert (wide == 9).all(), (kernel, pad)


FORMS = ["1,0"] + [f"{rows},{cut}" for rows in (64, 128, 256) for cut in (1, 2, 3, 4)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", [(1, 2560, 64), (70, 144, 320), (129, 1040, 832), (300, 4112, 256), (700, 272, 1984), (257, 2560, 1344)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_prefill_forms(shape, dtype, form, option):
    """The persistent form and every tile size and cut of the other, forced: whole and ragged tiles in both directions, fewer
    k-blocks than pairs asked for, more clusters than the GPU holds, any pitch; the oracle's bits, nothing written outside."""
    import torch
    M, K, N = shape
    t = getattr(torch, dtype)
    a, wp, rs, cs, ta, tw, trs, tcs = operands(M, K, N, M + N)
    c = oracle_lib.matmul(a, wp)
    bias = torch.randn(N, device="cuda")
    res = torch.randn(M, N, device="cuda").to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    option("fused_split", form)
    for pad in (0, 8, 3):
        for act, b, r in (("none", None, None), ("relu2", bias, res), ("relu", None, res), ("silu", bias, None)):
            wide = torch.full((M + 2, N + pad), 5.0, dtype=t, device="cuda")
            y = wide[1:M + 1, pad // 2:pad // 2 + N]
            if r is not None:
                y.copy_(r)                                       # in place, at the output's pitch
            tb.matmul_fused(ta, tw, trs, tcs, bias=b, activation=act, residual=y if r is not None else None, out=y, kernel="gemm_tc",
                            status=status)
            check(y, c, rs, cs[None, :], None if b is None else b.cpu().numpy(), act, None if r is None else r.float().cpu().numpy())
            y.fill_(5.0)
            assert (wide == 5).all()
    assert tb.last_launched_kernel() == ("ternary_gemm_tc3_kernel" if form == "1,0" else "ternary_gemm_split_kernel")
    assert int(status.item()) == 0


def test_residual_in_place():
    import torch
    for (M, K, N) in [(1, 2560, 2560), (20, 2560, 640), (50, 1024, 640), (300, 1040, 832), (7, 129, 132), (200, 3001, 1028)]:
        _, _, _, _, ta, tw, trs, _ = operands(M, K, N, 8)
        for pad in (0, 3):
            stream = torch.randn(M, N + pad, device="cuda").to(torch.bfloat16)[:, :N]
            want = tb.matmul_fused(ta, tw, trs, 0.1, residual=stream.clone())
            got = tb.matmul_fused(ta, tw, trs, 0.1, residual=stream, out=stream)
            assert got is stream and torch.equal(got, want)


def test_matches_matmul_dequant():
    """Without bias, activation and residual it is matmul_dequant, bit for bit."""
    import torch
    for (M, K, N) in [(1, 2560, 640), (30, 2560, 640), (300, 1040, 832), (7, 129, 132)]:
        _, _, _, _, ta, tw, trs, _ = operands(M, K, N, 2)
        assert torch.equal(tb.matmul_fused(ta, tw, trs, 0.0371), tb.matmul_dequant(ta, tw, trs, 0.0371))


def test_unaligned_operands():
    """A and W that start anywhere in memory (no TMA view): small problems directly, large ones through an aligned copy."""
    import torch
    for (M, K, N) in [(3, 64, 64), (1, 2560, 640), (200, 2560, 1024), (40, 4096, 2048)]:
        a, wp, rs, cs, ta, tw, trs, tcs = operands(M, K, N, 4)
        want = tb.matmul_fused(ta, tw, trs, tcs)
        ba = torch.empty(M * K + 3, dtype=torch.int8, device="cuda")
        bw = torch.empty(K * N // 4 + 5, dtype=torch.uint8, device="cuda")
        ua, uw = ba[3:].view(M, K), bw[5:].view(K, N // 4)
        ua.copy_(ta)
        uw.copy_(tw)
        assert torch.equal(tb.matmul_fused(ua, tw, trs, tcs), want)
        assert torch.equal(tb.matmul_fused(ta, uw, trs, tcs), want)
        assert torch.equal(tb.matmul_fused(ua, uw, trs, tcs), want)


def test_extreme_values_and_depth():
    """Sums at the ends of their range, K so deep that the scaled accumulators would overflow, scales and residuals that are
    not finite: a NaN or infinity stays in its own row, column or element."""
    import torch
    for (M, K, N) in [(2, 300000, 64), (2, 262144, 8), (1, 65536, 64), (20, 131072, 64)]:
        a = np.full((M, K), -128, dtype=np.int8)
        a[1:] = 127
        w = np.ones((K, N), dtype=np.int8)
        w[:, 1::2] = -1
        c = a.astype(np.int64) @ w.astype(np.int64)
        rs = np.linspace(0.5, 1.5, M).astype(F)
        y = tb.matmul_fused(torch.from_numpy(a).cuda(), torch.from_numpy(tb.pack_ternary(w)).cuda(), torch.from_numpy(rs).cuda(),
                            0.25, out_dtype=torch.float32)
        check(y, c, rs, F(0.25), None, "none", None)
    for (M, K, N) in [(4, 64, 64), (40, 256, 128), (100, 256, 320), (5, 33, 36)]:
        _, _, _, _, ta, tw, trs, tcs = operands(M, K, N, 6)
        res = torch.randn(M, N, device="cuda")
        want = {act: tb.matmul_fused(ta, tw, trs, tcs, activation=act, residual=res) for act in ACTS}
        trs2, tcs2, res2 = trs.clone(), tcs.clone(), res.clone()
        trs2[1] = float("nan")
        tcs2[3] = float("nan")
        res2[2, 5] = float("-inf")
        for act in ACTS:
            y = tb.matmul_fused(ta, tw, trs2, tcs2, activation=act, residual=res2)
            assert y[1].isnan().all() and y[:, 3].isnan().all() and y[2, 5] == float("-inf")
            keep = torch.ones(M, N, dtype=torch.bool, device="cuda")
            keep[1] = False
            keep[:, 3] = False
            keep[2, 5] = False
            assert torch.equal(y[keep], want[act][keep])


@pytest.mark.parametrize("M,N", [(1, 1 << 18), (24, 1 << 16), (300, 1 << 13)])
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(act, M, N):
    """Every activation from the smallest floats to the largest, through the bias of a product of zeros: the float64 function
    within its error (what rounds to zero or to its argument included), the limits at infinity, NaN."""
    import torch
    rng = np.random.default_rng(N)
    parts = [np.linspace(-30, 30, N // 2), np.geomspace(1e-38, 1e18, N // 8), -np.geomspace(1e-38, 1e18, N // 8),
             rng.normal(size=N - N // 2 - 2 * (N // 8) - 64) * 3, np.zeros(64)]
    v = np.concatenate(parts).astype(F)
    v[-4:] = [np.inf, -np.inf, np.nan, F(3e38) if act != "relu2" else F(1e19)]
    a, w = torch.zeros(M, 64, dtype=torch.int8, device="cuda"), torch.zeros(64, N // 4, dtype=torch.uint8, device="cuda")
    y = tb.matmul_fused(a, w, torch.ones(M, device="cuda"), 1.0, bias=torch.from_numpy(v).cuda(), activation=act, out_dtype=torch.float32)
    assert torch.equal(y[:1].expand_as(y).isnan(), y.isnan()) and torch.equal(y[:1].nan_to_num().expand_as(y), y.nan_to_num())
    got = y[0].cpu().numpy()
    end = [got[-4], got[-3], got[-2]]
    assert end[0] == np.inf and np.isnan(end[2])
    assert end[1] == (0 if act.startswith("relu") else -np.inf) if act in ("none", "relu", "relu2") else np.isnan(end[1])
    v, got = np.delete(v, [N - 4, N - 3, N - 2]), np.delete(got, [N - 4, N - 3, N - 2]).astype(np.float64)
    want = oracle.activate64(v, act)
    with np.errstate(over="ignore", invalid="ignore"):
        tol = oracle.activation_error(v, act)
    tol = np.nan_to_num(tol, nan=0.0) + np.abs(want) * 2.0 ** -24 + np.finfo(F).smallest_normal      # flushed to zero below it
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), (act, v[np.argmax(off)], got[np.argmax(off)], want[np.argmax(off)])


def test_empty_sizes():
    import torch
    a = torch.empty((3, 0), dtype=torch.int8, device="cuda")
    w = torch.empty((0, 16), dtype=torch.uint8, device="cuda")
    bias, res = torch.randn(64, device="cuda"), torch.randn(3, 64, device="cuda")
    rs = torch.ones(3, device="cuda")
    assert torch.equal(tb.matmul_fused(a, w, rs, 1.0, bias=bias, activation="relu", residual=res), bias.relu()[None, :] + res)
    assert (tb.matmul_fused(a, w, rs, 1.0) == 0).all()
    y = tb.matmul_fused(torch.empty((0, 64), dtype=torch.int8, device="cuda"), torch.zeros((64, 16), dtype=torch.uint8, device="cuda"),
                        torch.empty(0, device="cuda"), 1.0)
    assert y.shape == (0, 64)
    y = tb.matmul_fused(torch.zeros((3, 64), dtype=torch.int8, device="cuda"), torch.empty((64, 0), dtype=torch.uint8, device="cuda"), rs, 1.0)
    assert y.shape == (3, 0)


def test_output_past_32_bit_offsets():
    import torch
    M, K, N = 70000, 64, 32768
    a = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda")
    wp = tb.synth_packed_weights(K, N, 1)
    rs = torch.rand(M, device="cuda")
    y = tb.matmul_fused(a, torch.from_numpy(wp).cuda(), rs, 0.5)
    for rows in (slice(0, 40), slice(65520, 65560), slice(M - 40, M)):
        c = oracle_lib.matmul(a[rows].cpu().numpy(), wp)
        check(y[rows], c, rs[rows].cpu().numpy(), F(0.5), None, "none", None)


def test_streams_graphs_and_two_at_once():
    """On two streams at once (both may take scratch from the pool), and captured once and replayed on new inputs."""
    import torch
    shapes = [(1, 2560, 640), (20, 2560, 640), (50, 1024, 640), (300, 1040, 832), (7, 129, 132), (200, 3001, 1028)]
    ops = [operands(M, K, N, 10 + i)[4:] for i, (M, K, N) in enumerate(shapes)]
    want = [tb.matmul_fused(a, w, rs, cs, activation="silu") for a, w, rs, cs in ops]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = [tb.matmul_fused(a, w, rs, cs, activation="silu") for a, w, rs, cs in ops]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g in got for x, y in zip(g, want))
    graphs, outs = [], []
    for _ in range(2):                     # two graphs of the same calls, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([tb.matmul_fused(a, w, rs, cs, activation="silu") for a, w, rs, cs in ops])
        graphs.append(g)
    for seed in (1, 2):
        for a, *_ in ops:
            a.copy_(torch.from_numpy(tb.synth_activations(tuple(a.shape), seed)))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = [tb.matmul_fused(a, w, rs, cs, activation="silu") for a, w, rs, cs in ops]
        assert all(torch.equal(x, y) for o in outs for x, y in zip(o, want))


@pytest.mark.parametrize("M", [1, 5, 48, 300])
def test_feed_forward_block(M):
    """The operators as they are used: norm -> gate|up product -> gate -> down product onto the stream, against the same
    block in float64 on the codes and scales that each step really produced (one step's bound does not feed the next's)."""
    import torch
    D, FF = 640, 1728
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, D, generator=g, device="cuda").to(torch.bfloat16)
    stream = torch.randn(M, D, generator=g, device="cuda").to(torch.bfloat16)
    w_in, w_mid = torch.rand(D, device="cuda") + 0.5, torch.rand(FF, device="cuda") + 0.5
    wp_gu, wp_down = tb.synth_packed_weights(D, 2 * FF, 1), tb.synth_packed_weights(FF, D, 2)
    cs = torch.cat([torch.full((FF,), 0.04, device="cuda"), torch.full((FF,), 0.03, device="cuda")])
    q, s, h = tb.rmsnorm_quantize(x, w_in, residual=stream, eps=1e-5)
    gu = tb.matmul_fused(q, torch.from_numpy(wp_gu).cuda(), s, cs)
    q2, s2 = tb.glu_quantize(gu[:, :FF], gu[:, FF:], activation="relu2", weight=w_mid, eps=1e-5)
    y = tb.matmul_fused(q2, torch.from_numpy(wp_down).cuda(), s2, 0.02, residual=h)
    hf = h.float().cpu().numpy()
    assert torch.equal(h, (x.float() + stream.float()).to(torch.bfloat16))
    qr, m = oracle.quantize((hf * w_in.cpu().numpy()).astype(F))
    assert np.array_equal(q.cpu().numpy(), qr)
    check(gu, oracle_lib.matmul(qr, wp_gu), s.cpu().numpy(), cs.cpu().numpy()[None, :], None, "none", None)
    gf = gu.float().cpu().numpy()
    r = np.where(gf[:, :FF] < 0, F(0), gf[:, :FF])
    z = ((r * r).astype(F) * gf[:, FF:]).astype(F)
    q2r, m2 = oracle.quantize((z * w_mid.cpu().numpy()).astype(F))
    assert np.array_equal(q2.cpu().numpy(), q2r)
    check(y, oracle_lib.matmul(q2r, wp_down), s2.cpu().numpy(), F(0.02), None, "none", hf)
    # and against the block without any quantisation: each product's error is at most half a code step per summand
    W1, W2 = tb.unpack_ternary(wp_gu).astype(np.float64), tb.unpack_ternary(wp_down).astype(np.float64)
    ms = (hf.astype(np.float64) ** 2).mean(axis=1, keepdims=True)
    full = hf / np.sqrt(ms + 1e-5) * w_in.cpu().numpy()
    exact = (full @ W1) * cs.cpu().numpy()
    step = s.cpu().numpy()[:, None].astype(np.float64)
    # half a step per summand, the code's own fp32 rounding (127 x 3 x 2^-24 of a step), the scale's bound, one bfloat16 rounding
    bound = (0.5 + 127 * 3 * 2.0 ** -24) * step * np.abs(W1).sum(axis=0) * cs.cpu().numpy() + \
        np.abs(exact) * (2.0 ** -8 + 1e-5) + (np.abs(full) @ np.abs(W1)) * cs.cpu().numpy() * oracle.row_scale_bound(D) + 1e-6
    assert (np.abs(gf - exact) <= bound * (1 + 2.0 ** -8)).all()


def test_refusals():
    import torch
    _, _, _, _, a, w, rs, cs = operands(8, 64, 128, 1)
    r = torch.zeros(8, 128, dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: tb.matmul_fused(a.cpu(), w, rs, 1.0),
        lambda: tb.matmul_fused(a.float(), w, rs, 1.0),
        lambda: tb.matmul_fused(a, w.to(torch.int8), rs, 1.0),
        lambda: tb.matmul_fused(a[:, :32], w, rs, 1.0),
        lambda: tb.matmul_fused(a.t().contiguous().t(), w, rs, 1.0),
        lambda: tb.matmul_fused(a, w[:, ::2], rs, 1.0),
        lambda: tb.matmul_fused(a, w, rs[:7], 1.0),
        lambda: tb.matmul_fused(a, w, rs.double(), 1.0),
        lambda: tb.matmul_fused(a, w, rs.cpu(), 1.0),
        lambda: tb.matmul_fused(a, w, rs, cs[:127]),
        lambda: tb.matmul_fused(a, w, rs, cs.half()),
        lambda: tb.matmul_fused(a, w, rs, 1.0, bias=cs[:64]),
        lambda: tb.matmul_fused(a, w, rs, 1.0, bias=cs.double()),
        lambda: tb.matmul_fused(a, w, rs, 1.0, activation="tanh"),
        lambda: tb.matmul_fused(a, w, rs, 1.0, kernel="fast"),
        lambda: tb.matmul_fused(a, w, rs, 1.0, residual=r, out_dtype=torch.float32),
        lambda: tb.matmul_fused(a, w, rs, 1.0, residual=r[:4]),
        lambda: tb.matmul_fused(a, w, rs, 1.0, residual=r[:1].expand(8, 128)),
        lambda: tb.matmul_fused(a, w, rs, 1.0, out_dtype=torch.int32),
        lambda: tb.matmul_fused(a, w, rs, 1.0, out=r, out_dtype=torch.float16),
        lambda: tb.matmul_fused(a, w, rs, 1.0, out=r[:, :64]),
        lambda: tb.matmul_fused(a, w, rs, 1.0, out=torch.empty(128, 8, dtype=torch.bfloat16, device="cuda").t()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("M", [1, 6, 40, 200])
def test_back_to_back_without_waiting(M):
    """The layer kernels begin while the kernel before them still runs and wait for it before they touch memory: a chain
    that feeds itself in place, with torch's own kernels and a group launch between, gives the same bits queued in one go
    as with a synchronisation after every call."""
    import torch
    D, FF = 640, 1728
    w_gu, w_down = (torch.from_numpy(tb.synth_packed_weights(*s)).cuda() for s in ((D, 2 * FF, 1), (FF, D, 2)))
    gain = torch.rand(D, device="cuda") + 0.5
    group_a = torch.zeros(1, D, dtype=torch.int8, device="cuda")
    group_c = torch.zeros(1, 2 * FF, dtype=torch.int32, device="cuda")
    group = tb.ProjectionGroup([(group_a, w_gu, group_c)])

    def run(sync):
        done = torch.cuda.synchronize if sync else (lambda: None)
        g = torch.Generator(device="cuda").manual_seed(M)
        stream = torch.randn(M, D, generator=g, device="cuda").to(torch.bfloat16)
        x = torch.zeros_like(stream)
        q, s = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
        q2, s2 = torch.empty(M, FF, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
        gu = torch.empty(M, 2 * FF, dtype=torch.bfloat16, device="cuda")
        seen = []
        for step in range(60):
            tb.rmsnorm_quantize(x, gain, residual=stream, out=q, row_scale=s, residual_out=stream); done()
            tb.matmul_fused(q, w_gu, s, 0.05, out=gu); done()
            if step % 3 == 1:
                group_a.copy_(q[:1]); done()
                group.run(); done()
                seen.append(group_c.clone()); done()
            tb.glu_quantize(gu[:, :FF], gu[:, FF:], activation="silu", eps=1e-5, out=q2, row_scale=s2); done()
            tb.matmul_fused(q2, w_down, s2, 0.03, residual=x, out=x); done()
            if step % 4 == 2:
                x.mul_(0.5); done()
        torch.cuda.synchronize()
        return [stream, x, q, q2] + seen

    want, got = run(True), run(False)
    assert torch.isfinite(want[0]).all() and all(torch.equal(a, b) for a, b in zip(got, want))


def test_capture_across_streams():
    """A layer call whose predecessors in a captured graph lie on two streams, and one that two streams follow."""
    import torch
    _, _, _, _, a, w, rs, cs = operands(40, 1024, 640, 3)
    x = torch.randn(40, 1024, device="cuda").to(torch.bfloat16)
    r = torch.randn(40, 1024, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()

    def work(fork):
        main = torch.cuda.current_stream()
        y = x * 1
        if fork:
            side.wait_stream(main)
        with torch.cuda.stream(side if fork else main):
            z = r + 1
            q0, s0 = tb.rmsnorm_quantize(z)
        if fork:
            main.wait_stream(side)
        q, s, h = tb.rmsnorm_quantize(y, residual=z)
        if fork:
            side.wait_stream(main)
        with torch.cuda.stream(side if fork else main):
            o1 = tb.matmul_fused(q, w, s, cs)
        o2 = tb.matmul_fused(q0, w, s0, cs, activation="relu2")
        if fork:
            main.wait_stream(side)
        return q, s, h, o1, o2

    want = work(False)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = work(True)
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
