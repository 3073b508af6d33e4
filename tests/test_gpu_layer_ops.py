"""Norm and gate in front of the quantiser (rmsnorm_quantize, glu_quantize) on the GPU, against their CPU restatement: codes
and the residual stream bit for bit wherever every operation is exactly rounded, scales within the bound of an fp32 sum."""
import os
import sys

import numpy as np
import pytest

import ternixengine_b200 as tb

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import layer_ops_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16", "float32"]
# one element, less than a warp, whole vectors, odd lengths, every register form, beyond the registers of a CTA
SHAPES = [(1, 1), (3, 7), (2, 64), (1, 2560), (5, 2561), (37, 4099), (7, 4104), (4, 8192), (3, 16392), (2, 16401), (2, 32768), (2, 40968)]


def to_np(x):
    return x.float().cpu().numpy()


def make(shape, dtype, seed, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.rand(shape[0], 1, generator=g, device="cuda") * 8 + 0.01
    return (torch.randn(shape, generator=g, device="cuda") * rows * scale).to(getattr(torch, dtype))


def check_quantized(codes, scale, t32, ms, eps, K):
    """Codes equal the float32 restatement's bit for bit; scales within the bound, plus 2^-150: a float32 below 2^-126 is a
    multiple of 2^-149, so rounding to one is off by up to half of that whatever its relative size."""
    q, m = oracle.quantize(t32)
    assert np.array_equal(codes.cpu().numpy(), q)
    want = oracle.row_scale64(m, ms, eps)
    got = scale.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(got[ok] - want[ok]) <= want[ok] * oracle.row_scale_bound(K) + 2.0 ** -150).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm_quantize(shape, dtype, residual):
    import torch
    M, K = shape
    x = make(shape, dtype, M + K)
    x[M - 1] = 0 if M > 1 else x[M - 1]
    r = make(shape, dtype, M + K + 1, 3.0) if residual else None
    if residual and M > 1:
        r[M - 1] = 0
    for weight in (None, (torch.randn(K, device="cuda") * 0.3 + 1).to(x.dtype), torch.randn(K, device="cuda") * 0.3 + 1):
        got = tb.rmsnorm_quantize(x, weight, residual=r, eps=1e-5)
        h = to_np(x)
        if residual:
            h_t = (x.float() + r.float()).to(x.dtype)
            assert torch.equal(got[2], h_t)
            h = to_np(h_t)
        t = h if weight is None else (h * to_np(weight)[None, :]).astype(np.float32)
        check_quantized(got[0], got[1], t, (h.astype(np.float64) ** 2).mean(axis=1), 1e-5, K)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", list(tb.ACTIVATIONS))
def test_glu_quantize(shape, dtype, act):
    """relu, relu2 and none: bit for bit.  The others: a code lies within half a step and the activation's error of the
    exact quotient."""
    import torch
    M, K = shape
    gu = torch.cat([make(shape, dtype, K, 0.5), make(shape, dtype, K + 7)], dim=1)
    if M > 1:
        gu[M - 1] = 0
    gate, up = gu[:, :K], gu[:, K:]
    g, u = to_np(gate), to_np(up)
    for eps, weight in ((None, None), (1e-6, None), (1e-6, torch.randn(K, device="cuda") * 0.3 + 1)):
        codes, scale = tb.glu_quantize(gate, up, activation=act, weight=weight, eps=eps)
        w = np.ones(K, dtype=np.float32) if weight is None else to_np(weight)
        if act in ("none", "relu", "relu2"):
            a = g if act == "none" else np.where(g < 0, np.float32(0), g)
            a = (a * a).astype(np.float32) if act == "relu2" else a
            z = (a * u).astype(np.float32)
            t = z if weight is None else (z * w).astype(np.float32)
            check_quantized(codes, scale, t, (z.astype(np.float64) ** 2).mean(axis=1), eps, K)
            continue
        z = oracle.activate64(g, act) * u
        t = z * w
        # the activation's error, the roundings of act, act * up and * weight, and of the maximum
        err = (oracle.activation_error(g, act) + 3 * np.abs(oracle.activate64(g, act)) * 2.0 ** -24) * np.abs(u * w)
        m = np.abs(t).max(axis=1, keepdims=True)
        m_err = (err * (np.abs(t) + 2 * err >= m)).max(axis=1, keepdims=True)
        live = m[:, 0] > 0
        with np.errstate(all="ignore"):
            v = 127 * t / m
            bound = 0.5 + 127 * (err + np.abs(t) * m_err / m) / m + 127 * 3 * 2.0 ** -24
        q = codes.cpu().numpy().astype(np.float64)
        assert (np.abs(q - v)[live] <= bound[live]).all() and (q[~live] == 0).all()
        want = oracle.row_scale64(m[:, 0], (z ** 2).mean(axis=1), eps)
        # a norm's sum is off by at most twice the largest weighed error of its terms
        z_err = 2 * (err / np.maximum(np.abs(w), 1e-30) * np.abs(z)).sum(axis=1) / np.maximum((z ** 2).sum(axis=1), 1e-300)
        with np.errstate(all="ignore"):
            rel = oracle.row_scale_bound(K) + m_err[:, 0] / m[:, 0] + (0 if eps is None else z_err)
        got = scale.cpu().numpy().astype(np.float64)
        assert (np.abs(got - want)[live] <= (want * rel)[live]).all() and (got[~live] == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [2560, 2561, 40968])
def test_rows_that_are_not_ordinary(dtype, K):
    """Zeros, infinities, NaN, the type's lowest and smallest values, a sum of squares that leaves fp32, a single value."""
    import torch
    t = getattr(torch, dtype)
    info = torch.finfo(t)
    x = make((10, K), dtype, 5)
    x[0] = 0
    x[1, K // 2] = float("inf")
    x[2, K - 1] = float("-inf")
    x[3, 3] = float("nan")
    x[4] = info.min                              # float16: 65504^2 x K still fits fp32; the others overflow
    x[5] = info.smallest_normal * 2
    x[6] = 0
    x[6, K - 1] = -3.0
    x[7, 0] = float("inf")
    x[7, 1] = float("nan")
    x[8] = 0
    x[8, 5] = info.smallest_normal * info.eps if dtype == "float32" else info.smallest_normal     # smallest of all
    codes, scale = tb.rmsnorm_quantize(x, eps=1e-5)
    q, s = codes.cpu().numpy(), scale.cpu().numpy()
    bad = [1, 2, 3, 7] + ([4] if dtype != "float16" else [])
    assert (q[bad] == 0).all() and np.isnan(s[bad]).all()
    good = [i for i in range(10) if i not in bad]
    h = to_np(x)[good]
    check_quantized(codes[good], scale[good], h, (h.astype(np.float64) ** 2).mean(axis=1), 1e-5, K)
    assert s[0] == 1 and (q[5] == 127).all() and q[6, K - 1] == -127 and q[8, 5] == 127
    # the same rows as a gate's second factor: finite rows as before, the others poisoned, nothing spills into a neighbour
    one = torch.ones_like(x)
    cg, sg = tb.glu_quantize(one, x, activation="relu")
    bad = [1, 2, 3, 7]
    assert (cg.cpu().numpy()[bad] == 0).all() and np.isnan(sg.cpu().numpy()[bad]).all()
    good = [i for i in range(10) if i not in bad]
    check_quantized(cg[good], sg[good], to_np(x)[good], None, None, K)


def test_residual_in_place_and_pitches():
    """residual_out may be the residual or x; rows may have any pitch and start anywhere; what lies around stays.  Codes and
    h are the same bits; a scale may differ by twice its bound, because rows that a 16-byte load cannot address are spread
    over the threads in another order and each order's sum is within the bound of the exact one."""
    import torch

    def same(got, want):
        tol = 2 * oracle.row_scale_bound(got[0].shape[1])
        return torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and \
            bool(((got[1].double() - want[1].double()).abs() <= want[1].double() * tol).all())

    for dtype in (torch.bfloat16, torch.float32):
        for K, off, pad in ((2560, 0, 16), (2560, 3, 5), (130, 1, 2), (40970, 2, 6)):
            M = 6
            wide = torch.randn(M + 2, K + off + pad, device="cuda").to(dtype)
            res = torch.randn(M, K + pad, device="cuda").to(dtype)
            keep_w, keep_r = wide.clone(), res.clone()
            x, r = wide[1:M + 1, off:off + K], res[:, :K]
            want = tb.rmsnorm_quantize(x.contiguous(), residual=r.contiguous())
            got = tb.rmsnorm_quantize(x, residual=r)
            assert same(got, want)
            got = tb.rmsnorm_quantize(x, residual=r, residual_out=r)
            assert same(got, want) and got[2] is r
            assert torch.equal(res[:, K:], keep_r[:, K:]) and torch.equal(wide, keep_w)
            res.copy_(keep_r)
            got = tb.rmsnorm_quantize(x, residual=r, residual_out=x)
            assert same(got, want)
            wide[1:M + 1, off:off + K] = keep_w[1:M + 1, off:off + K]
            assert torch.equal(wide, keep_w) and torch.equal(res, keep_r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [297, 2961])
@pytest.mark.parametrize("vectors", [320, 321, 513, 1024, 1025, 2048, 2049, 4096])
def test_many_rows(dtype, M, vectors):
    """What is chosen by the number of rows: the rows as above in calls of fewer rows, where nothing of it runs.  Codes and h
    are the same bits; scales within twice the bound of a sum (another order).  Zero and poisoned rows between others, any
    pitch of whole vectors, the residual stream in place."""
    import torch
    t = getattr(torch, dtype)
    V = 4 if dtype == "float32" else 8
    K = vectors * V

    def pitched(seed, pad):
        return make((M, K + pad), dtype, seed)[:, :K]

    x, r, w = pitched(1, 2 * V), pitched(2, V), (torch.randn(K, device="cuda") * 0.3 + 1).to(t)
    x[5:M:97] = 0
    r[5:M:97] = 0
    x[11:M:131, K // 3] = float("nan")
    r[200, K - 1] = float("inf")
    tol = 2 * oracle.row_scale_bound(K)

    def same(got, pieces):
        for i, part in enumerate(pieces):
            rows = slice(100 * i, 100 * i + part[0].shape[0])
            assert torch.equal(got[0][rows], part[0])
            a, b = got[1][rows].double(), part[1].double()
            assert torch.equal(a.isnan(), b.isnan()) and bool(((a - b).abs() <= b * tol)[~b.isnan()].all())
            if len(got) == 3:
                assert torch.equal(got[2][rows].nan_to_num(nan=77.0), part[2].nan_to_num(nan=77.0))

    def pieces(f):
        return [f(slice(i, min(i + 100, M))) for i in range(0, M, 100)]

    same(tb.rmsnorm_quantize(x, w), pieces(lambda s: tb.rmsnorm_quantize(x[s], w)))
    want = pieces(lambda s: tb.glu_quantize(x[s], r[s], activation="silu", weight=w, eps=1e-5))
    same(tb.glu_quantize(x, r, activation="silu", weight=w, eps=1e-5), want)
    want = pieces(lambda s: tb.glu_quantize(x[s], r[s], activation="relu2"))
    same(tb.glu_quantize(x, r, activation="relu2"), want)
    want = pieces(lambda s: tb.rmsnorm_quantize(x[s], w, residual=r[s]))
    same(tb.rmsnorm_quantize(x, w, residual=r), want)
    got = tb.rmsnorm_quantize(x, w, residual=r, residual_out=r)
    assert got[2] is r
    same(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 8, 9, 32, 33, 64, 65])
@pytest.mark.parametrize("vectors", [513, 1025, 2049, 4096, 8191, 8193])
def test_a_few_long_rows(dtype, M, vectors):
    """Rows shared by the CTAs of a cluster (whole and partial shares, the last CTA with none), and what is next to them: too
    many rows for it, rows too long for it.  Zero rows, poisoned rows, the stream in place, any pitch of whole vectors."""
    import torch
    t = getattr(torch, dtype)
    V = 4 if dtype == "float32" else 8
    K = vectors * V
    x, r = make((M, K + V), dtype, M)[:, :K], make((M, K + 3 * V), dtype, M + 1)[:, :K]
    if M > 2:
        x[0], r[0] = 0, 0
        x[M - 1, K - 1] = float("nan")
    for weight in (None, (torch.randn(K, device="cuda") * 0.3 + 1).to(t), torch.randn(K, device="cuda") * 0.3 + 1):
        w = np.ones(K, dtype=np.float32) if weight is None else to_np(weight)
        codes, scale = tb.rmsnorm_quantize(x, weight)
        h = to_np(x)
        check_quantized(codes, scale, (h * w).astype(np.float32), (h.astype(np.float64) ** 2).mean(axis=1), 1e-5, K)
        z = (np.where(h < 0, np.float32(0), h) * to_np(r)).astype(np.float32)
        codes, scale = tb.glu_quantize(x, r, activation="relu", weight=weight, eps=None if weight is None else 1e-5)
        check_quantized(codes, scale, (z * w).astype(np.float32), (z.astype(np.float64) ** 2).mean(axis=1), None if weight is None else 1e-5, K)
        keep = r.clone()
        h_t = (x.float() + r.float()).to(t)
        codes, scale, h = tb.rmsnorm_quantize(x, weight, residual=r, residual_out=r)
        assert h is r and torch.equal(r.nan_to_num(nan=77.0), h_t.nan_to_num(nan=77.0))
        h = to_np(h_t)
        check_quantized(codes, scale, (h * w).astype(np.float32), (h.astype(np.float64) ** 2).mean(axis=1), 1e-5, K)
        r.copy_(keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [3, 150])
@pytest.mark.parametrize("K", [1, 5, 9, 641, 2561, 4099, 8191, 16375, 16401, 32761])
def test_rows_off_a_vector_boundary(dtype, M, K):
    """Odd rows without gaps (every operand equally far off a boundary), and every operand at an offset and pitch of its own;
    weights off a boundary in both types.  Nothing outside the rows is read into them or written."""
    import torch
    t = getattr(torch, dtype)
    nan = float("nan")

    def at(offset, pitch, values, fill):
        """`values` in rows of `pitch` from element `offset` of a buffer that holds `fill` otherwise."""
        flat = torch.full((offset + M * pitch + 16,), fill, dtype=values.dtype, device="cuda")
        view = flat[offset:offset + M * pitch].view(M, pitch)[:, :K]
        view.copy_(values)
        return flat, view

    x0, r0 = make((M, K), dtype, K), make((M, K), dtype, K + 1)
    w0 = torch.randn(K, device="cuda") * 0.3 + 1
    h0 = (x0.float() + r0.float()).to(t)
    ms = (to_np(h0).astype(np.float64) ** 2).mean(axis=1)
    for layout in (((0, K), (0, K), (0, K), 0, 0), ((1, K + 3), (2, K + 2), (3, K + 5), 1, 1), ((3, K), (0, K + 1), (5, K), 3, 2)):
        (xo, xp), (ro, rp), (ho, hp), qo, wo = layout
        for w_type in (None, torch.float32, t):
            w = None if w_type is None else torch.cat([torch.full((wo,), nan, device="cuda"), w0]).to(w_type)[wo:]
            (_, x), (_, r) = at(xo, xp, x0, nan), at(ro, rp, r0, nan)
            h_flat, h = at(ho, hp, torch.full_like(x0, 5), 5)
            q_flat = torch.full((M * K + 32,), 55, dtype=torch.int8, device="cuda")
            q, s = q_flat[qo:qo + M * K].view(M, K), torch.empty(M, device="cuda")
            tb.rmsnorm_quantize(x, w, residual=r, out=q, row_scale=s, residual_out=h)
            assert torch.equal(h, h0)
            v = to_np(h0) if w is None else (to_np(h0) * to_np(w)[None, :]).astype(np.float32)
            check_quantized(q, s, v, ms, 1e-5, K)
            h.fill_(5)
            assert (h_flat == 5).all()
            tb.rmsnorm_quantize(h0 if xo == 0 else at(xo, xp, h0, nan)[1], w, out=q, row_scale=s)
            check_quantized(q, s, v, ms, 1e-5, K)
            z = (np.where(to_np(x0) < 0, np.float32(0), to_np(x0)) * to_np(r0)).astype(np.float32)
            eps = None if w is None else 1e-5
            tb.glu_quantize(x, r, activation="relu", weight=w, eps=eps, out=q, row_scale=s)
            check_quantized(q, s, z if w is None else (z * to_np(w)[None, :]).astype(np.float32), (z.astype(np.float64) ** 2).mean(axis=1), eps, K)
            q.fill_(55)
            assert (q_flat == 55).all()
            want = tb.rmsnorm_quantize(x, w, residual=r)
            got = tb.rmsnorm_quantize(x, w, residual=r, residual_out=x)          # in place
            assert got[2] is x and torch.equal(x, h0) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_outputs_of_the_caller_and_empty_sizes():
    import torch
    x = make((9, 640), "bfloat16", 1)
    codes = torch.full((12, 640), 55, dtype=torch.int8, device="cuda")
    scale = torch.full((12,), 7.0, device="cuda")
    want = tb.rmsnorm_quantize(x)
    got = tb.rmsnorm_quantize(x, out=codes[:9], row_scale=scale[:9])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (codes[9:] == 55).all() and (scale[9:] == 7).all()
    empty = torch.empty((0, 640), dtype=torch.bfloat16, device="cuda")
    q, s = tb.rmsnorm_quantize(empty)
    assert q.shape == (0, 640) and s.shape == (0,)
    q, s = tb.rmsnorm_quantize(torch.empty((3, 0), dtype=torch.float32, device="cuda"))
    assert q.shape == (3, 0) and (s == 1).all()
    q, s, h = tb.rmsnorm_quantize(empty, residual=empty)
    assert h.shape == (0, 640)
    assert tb.glu_quantize(empty, empty)[0].shape == (0, 640)


def test_rows_past_32_bit_offsets():
    """Element offsets beyond 2^31 in the inputs and byte offsets beyond 2^31 in the codes."""
    import torch
    M, K = 66000, 32768
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    rows = [0, 65535, 65536, M - 1]
    x[rows] = make((4, K), "bfloat16", 3)
    codes, scale = tb.rmsnorm_quantize(x)
    h = to_np(x[rows])
    check_quantized(codes[rows], scale[rows], h, (h.astype(np.float64) ** 2).mean(axis=1), 1e-5, K)
    assert (codes[1:65535:977] == 0).all() and (scale[1:65535] == 1).all()


def test_streams_and_graphs():
    """On another stream, and captured once and replayed on new inputs."""
    import torch
    x, r = make((33, 2560), "bfloat16", 1), make((33, 2560), "bfloat16", 2)
    w = torch.randn(2560, device="cuda").to(torch.bfloat16)
    want = tb.rmsnorm_quantize(x, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tb.rmsnorm_quantize(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = tb.rmsnorm_quantize(x, w, residual=r)
        b = tb.glu_quantize(x, a[2], activation="silu", weight=w, eps=1e-5)
    for seed in (11, 12):
        x.copy_(make((33, 2560), "bfloat16", seed))
        g.replay()
        want = tb.rmsnorm_quantize(x, w, residual=r)
        want2 = tb.glu_quantize(x, want[2], activation="silu", weight=w, eps=1e-5)
        assert all(torch.equal(p, q) for p, q in zip(a, want)) and all(torch.equal(p, q) for p, q in zip(b, want2))


def test_refusals():
    import torch
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: tb.rmsnorm_quantize(x.cpu()),
        lambda: tb.rmsnorm_quantize(x.double()),
        lambda: tb.rmsnorm_quantize(x[0]),
        lambda: tb.rmsnorm_quantize(x.t()),
        lambda: tb.rmsnorm_quantize(x[:1].expand(4, 64)),
        lambda: tb.rmsnorm_quantize(x, w[:63]),
        lambda: tb.rmsnorm_quantize(x, w.half()),
        lambda: tb.rmsnorm_quantize(x, w.cpu()),
        lambda: tb.rmsnorm_quantize(x, residual=x.float()),
        lambda: tb.rmsnorm_quantize(x, residual=x[:3]),
        lambda: tb.rmsnorm_quantize(x, residual_out=x),
        lambda: tb.rmsnorm_quantize(x, eps=0.0),
        lambda: tb.rmsnorm_quantize(x, eps=float("nan")),
        lambda: tb.rmsnorm_quantize(x, eps=2.0),
        lambda: tb.rmsnorm_quantize(x, out=torch.empty((4, 64), dtype=torch.uint8, device="cuda")),
        lambda: tb.rmsnorm_quantize(x, out=torch.empty((4, 128), dtype=torch.int8, device="cuda")[:, :64]),
        lambda: tb.rmsnorm_quantize(x, row_scale=torch.empty(3, device="cuda")),
        lambda: tb.glu_quantize(x, x, activation="swish"),
        lambda: tb.glu_quantize(x, x, weight=w),
        lambda: tb.glu_quantize(x, x.half()),
        lambda: tb.glu_quantize(x, x[:, :32]),
        lambda: tb.glu_quantize(x, x, eps=0.0),
        lambda: tb.glu_quantize(x.cpu(), x.cpu()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
