"""Performance cases of the 8-bit integer operators, through the public entry
points of hymt2sharp_amd.HipBackend.

Four operators, the ones a prompt's layers run around attention when their
weights have 8-bit copies:

gemm     y[t][f] = ws[f] xs[t] sum_k x[t][k] w[f][k], w and x int8 codes, ws a
         scale per channel (weight row), xs one per token; y fp32, fp32 added
         to what is there (the residual), or bf16;
glu      act[t][f] = bf16(silu(g) u), g and u such products over the gate and
         the up rows;
norm     x += add (fp32, stored), then RMSNorm(x) gamma as int8 codes with a
         scale per row; without add x is read only;
rows     the rows of x (bf16 or fp32) as int8 codes with a scale per row.

A row's codes are rint(127 v / max|v|), ties to even, and its scale is
max|v| / 127; codes are returned as the values they stand for.

The shapes are the 32-layer model's (hidden 2048, FFN 6144, vocabulary 120818)
and, drawn, others around them.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN, FFN, VOCAB = 2048, 6144, 120818
EPS = 1e-6


def listed():
    return [
        # one token's o projection: the smallest product a step makes, launch and latency
        {"name": "gemm_1x2048x2048_f32", "kind": "gemm", "m": 1, "n": HIDDEN, "k": HIDDEN, "out": "f32"},
        # the output projection of one token: a stream of the whole weight, whose
        # rows are no multiple of 4
        {"name": "gemm_1x120818x2048_f32", "kind": "gemm", "m": 1, "n": VOCAB, "k": HIDDEN, "out": "f32"},
        # a sentence, the commonest prompt: down, added to the residual
        {"name": "gemm_61x2048x6144_acc", "kind": "gemm", "m": 61, "n": HIDDEN, "k": FFN, "out": "acc"},
        # a few paragraphs, a ragged length
        {"name": "gemm_700x2048x6144_bf16", "kind": "gemm", "m": 700, "n": HIDDEN, "k": FFN, "out": "bf16"},
        # o and down over a full prefill chunk
        {"name": "gemm_2048x2048x2048_bf16", "kind": "gemm", "m": 2048, "n": HIDDEN, "k": HIDDEN, "out": "bf16"},
        {"name": "gemm_2048x2048x6144_f32", "kind": "gemm", "m": 2048, "n": HIDDEN, "k": FFN, "out": "f32"},
        # gate/up with its SwiGLU: a sentence and a full chunk
        {"name": "glu_61x6144x2048", "kind": "glu", "m": 61, "n": FFN, "k": HIDDEN},
        {"name": "glu_2048x6144x2048", "kind": "glu", "m": 2048, "n": FFN, "k": HIDDEN},
        # the norm before a projection: one token, without an addition, and a
        # full chunk with the o projection's bf16 rows added
        {"name": "norm_1x2048", "kind": "norm", "m": 1, "n": HIDDEN, "add": "none"},
        {"name": "norm_2048x2048_add_bf16", "kind": "norm", "m": 2048, "n": HIDDEN, "add": "bf16"},
        # the attention's rows of a sentence, the SwiGLU's of a full chunk
        {"name": "rows_61x2048_f32", "kind": "rows", "m": 61, "n": HIDDEN, "io": "f32"},
        {"name": "rows_2048x6144_bf16", "kind": "rows", "m": 2048, "n": FFN, "io": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gemm", "gemm", "gemm", "gemm", "glu", "glu", "norm", "norm", "rows", "rows"])
    m = 1 if rng.random() < 0.15 else _log_int(rng, 2, 2048)
    if kind in ("norm", "rows"):
        n = 4 * _log_int(rng, 32, 2048)  # any multiple of 4 up to 8192
        if kind == "norm":
            return {"kind": kind, "m": m, "n": n, "add": rng.choice(["none", "bf16", "f32"])}
        return {"kind": kind, "m": m, "n": n, "io": rng.choice(["f32", "bf16"])}
    k = 128 * _log_int(rng, 2, 64)  # 256 to 8192
    n = _log_int(rng, 32, 12000 if kind == "gemm" else 8192)  # odd ones too
    # at most the largest listed case's operations
    m = max(1, min(m, 2048 * 2 * FFN * HIDDEN // ((2 if kind == "glu" else 1) * n * k)))
    if kind == "glu":
        return {"kind": kind, "m": m, "n": n, "k": k}
    return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["f32", "acc", "bf16"])}


# ---- inputs ------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _coded(v):
    """Rows of fp32 values as int8 codes and fp32 scales."""
    a = v.abs().amax(-1, keepdim=True)
    return torch.round(v * (127.0 / a)).to(torch.int8), (a / 127.0).squeeze(-1)


def _weight(g, n, k):
    """Weight rows: normal values of standard deviation 1 / sqrt(k)."""
    return _coded(_normal(g, n, k) / math.sqrt(k))


def _activations(g, m, n):
    """Rows as a transformer's are: normal, each row of its own size, and a
    few channels (one in 512) that are ten times larger in every row."""
    big = torch.where(torch.rand(n, generator=g, device="cuda") < 1 / 512, 10.0, 1.0)
    return _normal(g, m, n) * big * torch.exp(0.5 * _normal(g, m, 1))


_BACKEND = []


def _backend():
    """The program's one backend, and its stream for torch."""
    if not _BACKEND:
        from hymt2sharp_amd import HipBackend
        be = HipBackend(0)
        _BACKEND.extend([be, torch.cuda.ExternalStream(be.stream())])
    return _BACKEND


def prepare(case, seed):
    g = _gen(seed)
    m, n, kind = case["m"], case["n"], case["kind"]
    s = {"case": case}
    f32 = dict(device="cuda", dtype=torch.float32)
    if kind in ("gemm", "glu"):
        k = case["k"]
        s["w"], s["ws"] = _weight(g, n, k)
        if kind == "glu":
            s["up"], s["us"] = _weight(g, n, k)
        s["x"], s["xs"] = _coded(_activations(g, m, k))
        if kind == "gemm" and case["out"] == "acc":
            s["y0"] = _normal(g, m, n)
        half = kind == "glu" or case["out"] == "bf16"
        s["y"] = torch.empty(m, n, device="cuda", dtype=torch.bfloat16 if half else torch.float32)
    else:
        x = _activations(g, m, n)
        s["x"] = x.to(torch.bfloat16) if case.get("io") == "bf16" else x
        s["codes"] = torch.empty(m, n, device="cuda", dtype=torch.int8)
        s["scale"] = torch.empty(m, **f32)
        s["values"] = torch.empty(m, n, **f32)
        if kind == "norm":
            s["gamma"] = torch.rand(n, generator=g, **f32) * 0.2 + 0.9
            if case["add"] != "none":
                add = 0.3 * _activations(g, m, n)
                s["add"] = add.to(torch.bfloat16) if case["add"] == "bf16" else add
                s["h"] = torch.empty(m, n, **f32)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------


def _plain_product(w, ws, x, xs):
    return (x.float() @ w.float().t()) * ws * xs[:, None]


def _plain_codes(v):
    """Values of v's row codes, and max|v|; in 64 bits, which decide a code
    next to a border."""
    a = v.abs().amax(-1, keepdim=True)
    return torch.where(a > 0, torch.round(v * 127.0 / a), torch.zeros_like(v)), a


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "gemm":
        y = _plain_product(s["w"], s["ws"], s["x"], s["xs"])
        return y.to(torch.bfloat16) if c["out"] == "bf16" else s["y0"] + y if c["out"] == "acc" else y
    if kind == "glu":
        gate = _plain_product(s["w"], s["ws"], s["x"], s["xs"])
        up = _plain_product(s["up"], s["us"], s["x"], s["xs"])
        return (gate / (1.0 + torch.exp(-gate)) * up).to(torch.bfloat16)
    if kind == "rows":
        q, a = _plain_codes(s["x"].double())
        return [q.float() * (a / 127.0).float(), (a / 127.0).float().squeeze(-1)]
    h = s["x"] if c["add"] == "none" else s["x"] + s["add"].float()
    d = h.double()
    q, a = _plain_codes(d * s["gamma"].double())
    scale = (a / 127.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)).float()
    return [q.float() * scale, scale.squeeze(-1)] + ([] if c["add"] == "none" else [h])


def _ptr(t):
    return t.data_ptr()


def _calls(s):
    from hymt2sharp_amd import BF16, F32

    be, stream = _backend()
    c = s["case"]
    m, n, kind = c["m"], c["n"], c["kind"]
    if kind == "gemm":
        if c["out"] == "acc":
            with torch.cuda.stream(stream):  # the residual as the step before leaves it
                s["y"].copy_(s["y0"])
        be.gemm_i8(_ptr(s["w"]), _ptr(s["ws"]), n, c["k"], _ptr(s["x"]), _ptr(s["xs"]), m, _ptr(s["y"]),
                   accumulate=c["out"] == "acc", out_bf16=c["out"] == "bf16")
        return s["y"]
    if kind == "glu":
        be.gemm_i8_swiglu(_ptr(s["w"]), _ptr(s["ws"]), _ptr(s["up"]), _ptr(s["us"]), n, c["k"], _ptr(s["x"]),
                          _ptr(s["xs"]), m, _ptr(s["y"]))
        return s["y"]
    if kind == "rows":
        be.to_i8(_ptr(s["x"]), m, n, _ptr(s["codes"]), _ptr(s["scale"]), x_dtype=BF16 if c["io"] == "bf16" else F32)
    elif c["add"] == "none":
        be.rows_rmsnorm_i8(_ptr(s["x"]), m, n, _ptr(s["gamma"]), EPS, _ptr(s["codes"]), _ptr(s["scale"]))
    else:
        with torch.cuda.stream(stream):
            s["h"].copy_(s["x"])
        be.rows_rmsnorm_i8(_ptr(s["h"]), m, n, _ptr(s["gamma"]), EPS, _ptr(s["codes"]), _ptr(s["scale"]),
                           add=_ptr(s["add"]), add_dtype=BF16 if c["add"] == "bf16" else F32)
    with torch.cuda.stream(stream):  # the values that the codes stand for
        torch.mul(s["codes"], s["scale"][:, None], out=s["values"])
    return [s["values"], s["scale"]] + ([s["h"]] if "h" in s else [])


def run(state):
    return _calls(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    m, n, kind = case["m"], case["n"], case["kind"]
    if kind == "gemm":
        k = case["k"]
        out = {"f32": 4, "acc": 8, "bf16": 2}[case["out"]]
        return {"bytes": n * k + m * k + 4 * (n + m) + out * m * n, "flops": 2 * m * n * k}
    if kind == "glu":
        k = case["k"]
        return {"bytes": 2 * n * k + m * k + 4 * (2 * n + m) + 2 * m * n, "flops": 4 * m * n * k}
    if kind == "rows":
        return {"bytes": m * n * ((2 if case["io"] == "bf16" else 4) + 1) + 4 * m, "flops": 3 * m * n}
    add = {"none": 0, "bf16": 2 + 4, "f32": 4 + 4}[case["add"]]
    return {"bytes": m * n * (4 + 1 + add) + 4 * (m + n), "flops": 6 * m * n}


# ---- the same in 64 bits -----------------------------------------------------------


def _exact_product(codes, scales, x, xs):
    m, n = x.shape[0], codes.shape[0]
    y = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for f in range(0, n, 8192):  # a part of the channels at a time
        y[:, f:f + 8192] = torch.matmul(x.double(), codes[f:f + 8192].double().t().contiguous())
    return y.mul_(scales.double()).mul_(xs.double().unsqueeze(1))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "gemm":
        y = _exact_product(s["w"], s["ws"], s["x"], s["xs"])
        return y + s["y0"].double() if case["out"] == "acc" else y
    if kind == "glu":
        gate = _exact_product(s["w"], s["ws"], s["x"], s["xs"])
        return gate * torch.sigmoid(gate) * _exact_product(s["up"], s["us"], s["x"], s["xs"])
    if kind == "rows":
        v, root, h = s["x"].double(), 1.0, None
    else:
        h = s["x"].double()
        if "add" in s:  # the sum is stored, and normed, as an fp32 value
            h = (h + s["add"].double()).float().double()
        v = h * s["gamma"].double()
        root = (h.square().sum(-1) / case["n"] + EPS).sqrt()
    top = torch.maximum(v.max(-1).values, -v.min(-1).values)
    codes = (127.0 * v).div(top.unsqueeze(1)).round()
    scale = top / (127.0 * root)
    return [codes * scale.unsqueeze(1), scale] + ([h] if kind == "norm" and "add" in s else [])
