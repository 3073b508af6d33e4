"""The operators around the ternary product, as cases to measure: what a quantised layer does before and after
C[M,N] = A[M,K] x W[K,N].

  rmsnorm_quantize   residual addition, root-mean-square norm, int8 activations with one scale per row
  matmul_fused       the product with scales, bias, activation and residual in its epilogue
  glu_quantize       gated activation (with or without a norm behind it), int8 activations with one scale per row

`run` computes them from elementary torch operations, or, where `own` is true, with the package's entry points.  The int8
activations are returned as the values they stand for (code x row scale), in bfloat16: its eight significant bits hold
every code.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one token of a 2560-wide model: what stands between two of its products
        {"name": "norm_token", "op": "norm", "m": 1, "k": 2560, "dtype": "bf16", "residual": True},
        # a ragged batch with an odd row length (no vector of a row is aligned)
        {"name": "norm_ragged", "op": "norm", "m": 333, "k": 2561, "dtype": "f16", "residual": True},
        # first norm of a model that keeps its stream in float32: nothing to add yet
        {"name": "norm_f32", "op": "norm", "m": 512, "k": 4096, "dtype": "f32", "residual": False},
        # prefill of 4096 tokens, 8192 wide
        {"name": "norm_prefill", "op": "norm", "m": 4096, "k": 8192, "dtype": "bf16", "residual": True},
        # one token through the feed-forward block of a 2560-wide model: squared ReLU gate and the norm behind it
        {"name": "glu_token", "op": "glu", "m": 1, "k": 6912, "dtype": "bf16", "act": "relu2", "norm": True},
        # the same for a prompt of 256 tokens
        {"name": "glu_prompt", "op": "glu", "m": 256, "k": 6912, "dtype": "bf16", "act": "relu2", "norm": True},
        # prefill of 4096 tokens, 28672 wide, SiLU gate straight into the quantiser
        {"name": "glu_prefill", "op": "glu", "m": 4096, "k": 28672, "dtype": "bf16", "act": "silu", "norm": False},
        # one token, output projection of a 2560-wide model added to its residual stream
        {"name": "mm_token", "op": "mm", "m": 1, "k": 2560, "n": 2560, "dtype": "bf16", "act": "none", "bias": False,
         "residual": True, "col_scale": False},
        # 32 sequences in decode, 4096 -> 11008 with bias and SiLU
        {"name": "mm_batch", "op": "mm", "m": 32, "k": 4096, "n": 11008, "dtype": "f16", "act": "silu", "bias": True,
         "residual": False, "col_scale": True},
        # a batch whose sizes no aligned copy fits
        {"name": "mm_ragged", "op": "mm", "m": 129, "k": 1029, "n": 2052, "dtype": "f32", "act": "gelu", "bias": True,
         "residual": True, "col_scale": False},
        # a prompt of 256 tokens, down projection of a 2560-wide model added to its residual stream
        {"name": "mm_prompt", "op": "mm", "m": 256, "k": 6912, "n": 2560, "dtype": "bf16", "act": "none", "bias": False,
         "residual": True, "col_scale": False},
        # prefill of 4096 tokens, 8192 -> 28672 with bias and squared ReLU
        {"name": "mm_prefill", "op": "mm", "m": 4096, "k": 8192, "n": 28672, "dtype": "bf16", "act": "relu2", "bias": True,
         "residual": False, "col_scale": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "glu", "mm"])
    m = _log_int(rng, 1, 4096)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    ragged = rng.random() < 0.25
    if op == "norm":
        k = _log_int(rng, 64, 8192)
        return {"op": op, "m": m, "k": k if ragged else -(-k // 16) * 16, "dtype": dtype, "residual": rng.random() < 0.7}
    if op == "glu":
        k = _log_int(rng, 64, 28672)
        return {"op": op, "m": m, "k": k if ragged else -(-k // 16) * 16, "dtype": "bf16" if dtype == "f32" and m * k > 1 << 25 else dtype,
                "act": rng.choice(["relu2", "silu", "gelu"]), "norm": rng.random() < 0.6}
    k, n = _log_int(rng, 64, 8192), _log_int(rng, 64, 28672)
    if ragged:      # no wider than a product that an unaligned model has: the largest is an aligned one
        m, n = min(m, 1024), -(-min(n, 8192) // 4) * 4
    else:
        k, n = -(-k // 16) * 16, -(-n // 64) * 64
    return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": rng.choice(["none", "relu2", "silu", "gelu"]),
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "col_scale": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, t = "cuda", _DTYPES[case["dtype"]]
    m, k = case["m"], case["k"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": dict(case), "eps": 1e-5}
    if case["op"] == "mm":
        n = case["n"]
        s["a"] = (normal(m, k) * 32).round_().clamp_(-127, 127).to(torch.int8)
        # iid weights, P(0) = 0.4 and P(-1) = P(+1) = 0.3, packed four to a byte along the columns (0 -> 0, +1 -> 1, -1 -> 3)
        packed = torch.zeros(k, n // 4, dtype=torch.uint8, device=dev)
        for j in range(4):
            u = torch.rand(k, n // 4, generator=g, device=dev)
            packed |= ((u > 0.4).to(torch.uint8) + 2 * (u > 0.7).to(torch.uint8)) << (2 * j)
        s["w"] = packed
        s["row_scale"] = torch.rand(m, generator=g, device=dev) * 0.02 + 0.002
        s["w_scale"] = torch.rand(n, generator=g, device=dev) * 0.05 + 0.02 if case["col_scale"] else 0.0371
        s["bias"] = normal(n) if case["bias"] else None
        s["residual"] = normal(m, n).to(t) if case["residual"] else None
        s["out"] = torch.empty(m, n, dtype=t, device=dev)
        return s
    s["codes"] = torch.empty(m, k, dtype=torch.int8, device=dev)
    s["scale"] = torch.empty(m, dtype=torch.float32, device=dev)
    s["values"] = torch.empty(m, k, dtype=torch.bfloat16, device=dev)
    channel = torch.exp(normal(k) * 0.5)                                   # some channels are larger than others
    s["weight"] = (1 + 0.2 * normal(k)).to(t)
    if case["op"] == "norm":
        x = normal(m, k) * channel
        if m > 4:
            x[m - 1] = 0                                                   # a padded row
        s["x"] = x.to(t)
        if case["residual"]:
            r = normal(m, k) * channel * 3
            if m > 4:
                r[m - 1] = 0
            s["residual"], s["h"] = r.to(t), torch.empty(m, k, dtype=t, device=dev)
        return s
    # gate and up lie side by side, as one product over both weight matrices leaves them
    gu = torch.empty(m, 2 * k, dtype=t, device=dev)
    gu[:, :k] = normal(m, k)
    gu[:, k:] = normal(m, k) * channel
    if m > 4:
        gu[m - 1] = 0
    s["gu"] = gu
    return s


def _activation(x, act):
    if act == "relu2":
        r = torch.relu(x)
        return r * r
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _quantize(t, norm, codes_out, scale_out):
    """Row by row: codes rint(t x 127 / absmax) and scales absmax / 127 x norm; rows of zeros have scale 1."""
    top = t.abs().amax(dim=1)
    some = top > 0
    codes = torch.round(t * torch.where(some, 127.0 / top, torch.zeros_like(top))[:, None])
    scale = torch.where(some, top / 127.0 * norm, torch.ones_like(top))
    codes_out.copy_(codes)
    scale_out.copy_(scale)
    return scale


def _values(s):
    return torch.mul(s["codes"], s["scale"][:, None], out=s["values"])


def _plain(s):
    case, eps = s["case"], s["eps"]
    if case["op"] == "mm":
        shifts = torch.arange(0, 8, 2, dtype=torch.uint8, device=s["w"].device)
        field = (s["w"].unsqueeze(-1) >> shifts).view(case["k"], case["n"])
        w = (field & 1).float() - (field & 2).float()
        y = s["a"].float() @ w
        y = (y * s["row_scale"][:, None]) * s["w_scale"]
        if s["bias"] is not None:
            y = y + s["bias"]
        y = _activation(y, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        s["out"].copy_(y)
        return {"y": s["out"]}
    if case["op"] == "norm":
        h = s["x"].float()
        if case["residual"]:
            s["h"].copy_(h + s["residual"].float())
            h = s["h"].float()
        norm = 1 / torch.sqrt(h.square().mean(dim=1) + eps)
        _quantize(h * s["weight"].float(), norm, s["codes"], s["scale"])
        out = {"values": _values(s), "scale": s["scale"]}
        if case["residual"]:
            out["h"] = s["h"]
        return out
    k = case["k"]
    z = _activation(s["gu"][:, :k].float(), case["act"]) * s["gu"][:, k:].float()
    norm = 1.0
    if case["norm"]:
        norm = 1 / torch.sqrt(z.square().mean(dim=1) + eps)
        z = z * s["weight"].float()
    _quantize(z, norm, s["codes"], s["scale"])
    return {"values": _values(s), "scale": s["scale"]}


def run(s):
    if not own:
        return _plain(s)
    import ternixengine_b200 as tb

    case = s["case"]
    if case["op"] == "mm":
        return {"y": tb.matmul_fused(s["a"], s["w"], s["row_scale"], s["w_scale"], bias=s["bias"], activation=case["act"],
                                     residual=s["residual"], out=s["out"])}
    if case["op"] == "norm":
        if case["residual"]:
            tb.rmsnorm_quantize(s["x"], s["weight"], residual=s["residual"], eps=s["eps"], out=s["codes"],
                                row_scale=s["scale"], residual_out=s["h"])
            return {"values": _values(s), "scale": s["scale"], "h": s["h"]}
        tb.rmsnorm_quantize(s["x"], s["weight"], eps=s["eps"], out=s["codes"], row_scale=s["scale"])
        return {"values": _values(s), "scale": s["scale"]}
    k = case["k"]
    gate, up = s["gu"][:, :k], s["gu"][:, k:]
    if case["norm"]:
        tb.glu_quantize(gate, up, activation=case["act"], weight=s["weight"], eps=s["eps"], out=s["codes"],
                        row_scale=s["scale"])
    else:
        tb.glu_quantize(gate, up, activation=case["act"], out=s["codes"], row_scale=s["scale"])
    return {"values": _values(s), "scale": s["scale"]}


def work(case):
    m, k, e = case["m"], case["k"], _BYTES[case["dtype"]]
    if case["op"] == "mm":
        n = case["n"]
        b = m * k + k * n // 4 + m * n * e + 4 * m
        b += 4 * n * (case["bias"] + case["col_scale"]) + m * n * e * case["residual"]
        return {"bytes": b, "flops": 2 * m * k * n}
    values = 2 * m * k + 4 * m                      # the values that the codes stand for, and the scales
    if case["op"] == "norm":
        return {"bytes": m * k * e * (3 if case["residual"] else 1) + k * e + values + m * k, "flops": 8 * m * k}
    return {"bytes": 2 * m * k * e + k * e * case["norm"] + values + m * k, "flops": 12 * m * k}


# ---- the same in 64 bits, from the definitions

_ERF = np.vectorize(math.erf, otypes=[np.float64])


def _act64(v, act):
    if act == "relu2":
        return torch.where(v > 0, v * v, torch.zeros_like(v))
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        if v.numel() <= 1 << 18:
            return torch.from_numpy(v.cpu().numpy() * (1 + _ERF(v.cpu().numpy() / math.sqrt(2))) / 2).to(v.device)
        return v * torch.special.ndtr(v)
    return v


def _codes64(t, norm):
    top = torch.linalg.vector_norm(t, ord=math.inf, dim=1, keepdim=True)
    live = top > 0
    step = torch.where(live, top / 127, torch.ones_like(top))
    values = torch.round(t / step) * step * norm
    return {"values": values, "scale": torch.where(live, step * norm, torch.ones_like(top)).squeeze(1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "mm":
        code = torch.stack([s["w"].bitwise_right_shift(2 * j).bitwise_and(3) for j in range(4)], dim=2).flatten(1)
        table = torch.tensor([0.0, 1.0, math.nan, -1.0], dtype=torch.float64, device=code.device)
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=code.device)
        a = s["a"].double()
        for lo in range(0, case["n"], 4096):
            y[:, lo:lo + 4096] = a @ table[code[:, lo:lo + 4096].int()]
        y = torch.einsum("mn,m->mn", y, s["row_scale"].double())
        y = y * (s["w_scale"].double() if case["col_scale"] else float(np.float32(s["w_scale"])))
        if case["bias"]:
            y += s["bias"].double()
        y = _act64(y, case["act"])
        if case["residual"]:
            y += s["residual"].double()
        return {"y": y}
    if case["op"] == "norm":
        h = s["x"].double()
        if case["residual"]:
            # the stream is held in the inputs' type: the norm reads what was rounded to it
            total = h + s["residual"].double()
            h = total.to(s["x"].dtype).double()
        ms = (h * h).sum(dim=1, keepdim=True) / case["k"]
        out = _codes64(h * s["weight"].double(), (ms + s["eps"]) ** -0.5)
        if case["residual"]:
            out["h"] = total
        return out
    gate, up = s["gu"].double().split(case["k"], dim=1)
    z = _act64(gate, case["act"]) * up
    if not case["norm"]:
        return _codes64(z, 1.0)
    ms = (z * z).sum(dim=1, keepdim=True) / case["k"]
    return _codes64(z * s["weight"].double(), (ms + s["eps"]) ** -0.5)
