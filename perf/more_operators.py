"""Performance cases of the multi-sequence cache's operators, through the public
entry points of hymt2sharp_amd.HipBackend.

Many sequences share one pool of pages of 64 positions; a sequence is a slot with
a row of the page table and a length, and several may hold the same page.  Four
operators serve a batch of them:

pages    the pool's upkeep.  fork: child slots take their parents' pages, a page
         that the sequence ends inside as a copy; extend: room for new
         positions, lengths grow; compact: the pages in use move to the front
         of the pool;
rope     rotary positions, RMSNorm per head and append: q rows out, k and v rows
         into their pages;
packed   causal attention of packed prompts of different lengths over the pages;
shared   attention of one row per sequence where all sequences begin with the
         same prefix, read once for all of them.

A page of one kv head holds its 64 positions in 16-byte chunks of 8 values:
K chunk (s, j, c) = dims 8 j .. 8 j + 7 of position 16 s + c at chunk
(s D / 8 + j) 16 + c, V chunk (4 m + g, d) = dim d of positions 32 m + 4 g + [0, 4)
and 32 m + 16 + 4 g + [0, 4) at chunk (4 m + g) D + d.

Lengths of a case are drawn from its own numbers (`mix`), not from the seed.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 64
EPS = 1e-6
BASE = 10000.0


def listed():
    model = {"hkv": 4, "group": 4, "d": 128}
    return [
        # a decode step of 64 requests: a new position each, a page for few of them
        {"name": "pages_extend_64", "kind": "pages", "op": "extend", "n": 64, "lo": 30, "hi": 4000, "layers": 2,
         "mix": 1, "pages": 2400, **model},
        # a beam of 16 from one request: its last page, copied in all 32 layers
        {"name": "pages_fork_16", "kind": "pages", "op": "fork", "n": 16, "lo": 1000, "hi": 1000, "layers": 32,
         "mix": 2, "pages": 64, **model},
        # a fragmented pool after a burst of requests
        {"name": "pages_compact_512", "kind": "pages", "op": "compact", "n": 24, "lo": 500, "hi": 1400, "layers": 8,
         "mix": 3, "pages": 512, "moved": 150, **model},
        # the rows of a decode step, at far and near positions
        {"name": "rope_decode_64", "kind": "rope", "n": 64, "lo": 1, "hi": 1, "past_lo": 1, "past_hi": 30000, "mix": 4,
         "pad": 0, "rot": 128, "pairs": "half", "scaling": "none", "norm": True, "io": "f32", "dtype": "bf16", **model},
        # packed prompts, half of each head rotated, contexts stretched four times
        {"name": "rope_prompts_16k", "kind": "rope", "n": 9, "lo": 300, "hi": 4096, "past_lo": 0, "past_hi": 0, "mix": 5,
         "pad": 37, "rot": 64, "pairs": "interleaved", "scaling": "yarn", "norm": True, "io": "bf16", "dtype": "f16",
         **model},
        # sentences, the commonest request
        {"name": "packed_32_sentences", "kind": "packed", "n": 32, "lo": 4, "hi": 128, "past_lo": 0, "past_hi": 0,
         "mix": 6, "pad": 0, "dtype": "bf16", **model},
        # prompts from a word to a document together, one of them empty
        {"name": "packed_9_to_2048", "kind": "packed", "n": 9, "lo": 0, "hi": 2048, "past_lo": 0, "past_hi": 0,
         "mix": 7, "pad": 5, "dtype": "f16", **model},
        # chunks of 256 over 8192 cached positions
        {"name": "packed_2x256_at_8192", "kind": "packed", "n": 2, "lo": 256, "hi": 256, "past_lo": 8192,
         "past_hi": 8192, "mix": 8, "pad": 0, "dtype": "f16", **model},
        # whole documents
        {"name": "packed_4_to_8192", "kind": "packed", "n": 4, "lo": 4096, "hi": 8192, "past_lo": 0, "past_hi": 0,
         "mix": 9, "pad": 0, "dtype": "bf16", **model},
        # a few requests behind a short instruction
        {"name": "shared_8_at_512", "kind": "shared", "n": 8, "prefix": 512, "lo": 1, "hi": 64, "mix": 10,
         "dtype": "bf16", **model},
        # a server's batch behind a long instruction with examples
        {"name": "shared_64_at_4096", "kind": "shared", "n": 64, "prefix": 4096, "lo": 1, "hi": 512, "mix": 11,
         "dtype": "bf16", **model},
        # many questions about one long document
        {"name": "shared_256_at_16384", "kind": "shared", "n": 256, "prefix": 16384, "lo": 64, "hi": 1024, "mix": 12,
         "dtype": "f16", **model},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv, group = rng.choice([(4, 4), (4, 4), (1, 8), (2, 7), (8, 1), (8, 4), (3, 5), (2, 16), (5, 2)])
    return {"hkv": hkv, "group": group, "d": rng.choice([128, 128, 64])}


def _fitted(case):
    """Fewer sequences, or a shorter one, until a case costs no more than the largest
    listed one and its pages fit in 512 MB."""
    while (work(case)["flops"] > 4e11 or
           _pages_of(case) * case["hkv"] * PAGE * case["d"] * 4 > 1 << 29):
        if case["n"] > 1:
            case["n"] = (case["n"] + 1) // 2
        else:
            case["hi"] = max(case["hi"] // 2, 1)
            case["past_hi"] = max(case["past_hi"] // 2, case["past_lo"])
    return case


def draw(rng):
    kind = rng.choice(["pages", "rope", "rope", "packed", "packed", "packed", "shared", "shared", "shared"])
    mix = rng.randrange(1 << 30)
    h = _heads(rng)
    if kind == "pages":
        op = rng.choice(["extend", "fork", "compact"])
        n = _log_int(rng, 1, 128)
        lo = _log_int(rng, 1, 500)
        hi = lo + _log_int(rng, 1, 1000)
        layers = _log_int(rng, 1, 8)
        pages = n * (hi // PAGE + 3) * (2 if op == "fork" else 1) + rng.randrange(20)
        # at most 1 GB of pages
        layers = max(1, min(layers, (1 << 30) // (pages * h["hkv"] * PAGE * h["d"] * 4)))
        c = {"kind": kind, "op": op, "n": n, "lo": lo, "hi": hi, "layers": layers, "mix": mix, "pages": pages, **h}
        if op == "compact":
            c["moved"] = rng.randrange(pages - _pages_of(c) + 1)
        return c
    if kind == "rope":
        one = rng.random() < 0.4
        lo = 1 if one else rng.randrange(3)
        hi = 1 if one else _log_int(rng, 4, 2000)
        past_hi = _log_int(rng, 1, 30000) if rng.random() < 0.6 else 0
        n = _log_int(rng, 1, 256 if one else 16)
        return _fitted(
            {"kind": kind, "n": n, "lo": lo, "hi": hi, "past_lo": min(1, past_hi), "past_hi": past_hi, "mix": mix,
             "pad": rng.choice([0, 0, 3, 60]), "rot": rng.choice([0, 16, 32, 48, 64] + [h["d"]] * 3),
             "pairs": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
             "norm": rng.random() < 0.7, "io": rng.choice(["f32", "bf16", "f16"]), "dtype": rng.choice(["f16", "bf16"]),
             **h})
    if kind == "packed":
        n = _log_int(rng, 1, 40)
        hi = _log_int(rng, 2, 4096 if n <= 8 else 800)
        past_hi = _log_int(rng, 1, 6000) if rng.random() < 0.4 else 0
        return _fitted(
            {"kind": kind, "n": n, "lo": rng.randrange(3), "hi": hi, "past_lo": min(1, past_hi), "past_hi": past_hi,
             "mix": mix, "pad": rng.choice([0, 0, 1, 40]), "dtype": rng.choice(["f16", "bf16"]), **h})
    prefix = PAGE * (0 if rng.random() < 0.15 else _log_int(rng, 1, 256))
    n = _log_int(rng, 1, 256)
    return {"kind": kind, "n": n, "prefix": prefix, "lo": 1, "hi": _log_int(rng, 2, 1024), "mix": mix,
            "dtype": rng.choice(["f16", "bf16"]), **h}


# ---- lengths -----------------------------------------------------------------------


def _spread(rng, lo, hi, n):
    """n lengths from lo to hi, even over their logarithm, the first lo and the last hi."""
    v = [int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 for _ in range(n)]
    if n > 1:
        v[0] = lo
    v[-1] = hi
    rng.shuffle(v)
    return v


def _lens(case):
    """(new positions, length with them) of each sequence."""
    rng = random.Random(case["mix"])
    n, kind = case["n"], case["kind"]
    if kind == "pages":
        cur = _spread(rng, case["lo"], case["hi"], n)
        if case["op"] == "fork" and n > 1:  # one request forks: every entry has its length
            cur = [cur[0]] * n
        return [1] * n, cur
    new = [1] * n if kind == "shared" else _spread(rng, case["lo"], case["hi"], n)
    if kind == "shared":
        return new, [case["prefix"] + k for k in _spread(rng, case["lo"], case["hi"], n)]
    past = _spread(rng, case["past_lo"], case["past_hi"], n)
    return new, [a + b for a, b in zip(new, past)]


def _blocks(length):
    return -(-length // PAGE)


def _pages_of(case):
    """Pages that the case's sequences hold before the pass."""
    _, lens = _lens(case)
    if case["kind"] == "pages" and case["op"] == "fork":
        return _blocks(lens[0])
    shared = case.get("prefix", 0) // PAGE
    return shared + sum(_blocks(k) - shared for k in lens)


# ---- inputs ------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(d):
    """Element offsets [64][d] of a position and dim in a K and in a V page."""
    t = torch.arange(PAGE, device="cuda").view(-1, 1)
    i = torch.arange(d, device="cuda").view(1, -1)
    ko = ((t // 16 * (d // 8) + i // 8) * 16 + t % 16) * 8 + i % 8
    vo = ((4 * (t // 32) + t // 4 % 4) * d + i) * 8 + 4 * (t // 16 % 2) + t % 4
    return ko, vo


def _frequencies(case):
    """Radians per position of each pair, and the factor on cosine and sine."""
    rot, factor, trained = case["rot"], 4.0, 4096
    base = BASE
    if case["scaling"] == "ntk" and rot > 2:
        base = BASE * factor ** (rot / (rot - 2))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if case["scaling"] == "linear":
        f = [x / factor for x in f]
    if case["scaling"] != "yarn" or rot == 0:
        return f, 1.0

    def dim_of(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo = max(math.floor(dim_of(32.0)), 0)
    hi = min(math.ceil(dim_of(1.0)), rot - 1)
    out = []
    for i, x in enumerate(f):
        r = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
        out.append(x / factor * r + x * (1.0 - r))
    return out, 0.1 * math.log(factor) + 1.0


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
    kind, n = case["kind"], case["n"]
    hkv, group, d = case["hkv"], case["group"], case["d"]
    new, lens = _lens(case)
    cells = hkv * PAGE * d
    s = {"case": case, "new": new, "lens": lens, "layer": 0}
    perm = random.Random(int(seed) * 7919 + case["mix"])

    # the sequences' pages, anywhere in the pool
    seqs = 2 * n + 3
    grown = [k + (1 if kind == "pages" else 0) for k in lens]
    blocks = max(_blocks(k) for k in grown) + 2
    table = np.full((seqs, blocks), -1, np.int32)
    held = np.zeros(seqs, np.int32)
    if kind == "pages":
        dtype, layers, pages = torch.bfloat16, case["layers"], case["pages"]
        live = _pages_of(case)
        if case["op"] == "compact":
            m = min(case["moved"], live, pages - live)
            s["moved"] = m
            holes = set(perm.sample(range(live), m))
            front = [p for p in range(live) if p not in holes] + perm.sample(range(live, pages), m)
        else:
            front = perm.sample(range(pages), live)
    else:
        dtype, layers = _TYPES[case["dtype"]], 1
        live = _pages_of(case)
        pages = live + 3
        front = perm.sample(range(pages), live)
    perm.shuffle(front)
    order = perm.sample(range(seqs), 2 * n)
    slots = order[:n]
    prefix = case.get("prefix", 0) // PAGE
    used = 0
    for i in range(1 if kind == "pages" and case["op"] == "fork" else n):
        nb = _blocks(lens[i])
        first = prefix if i > 0 else 0  # the prefix's pages are the first sequence's
        table[slots[i], :first] = table[slots[0], :first]
        table[slots[i], first:nb] = front[used:used + nb - first]
        held[slots[i]] = lens[i]
        used += nb - first
    refs = np.zeros(pages, np.int32)
    for r in range(seqs):
        for p in table[r, :_blocks(int(held[r]))]:
            refs[p] += 1
    # one buffer of whole numbers: table, lengths, references and the operators' own room
    sizes = [seqs * blocks, seqs, pages, 4 + 3 * pages]
    meta = np.concatenate([table.reshape(-1), held, refs, np.zeros(sizes[3], np.int32)])
    s["meta0"] = torch.from_numpy(meta).cuda()
    s["meta"] = s["meta0"].clone()
    parts = torch.split(s["meta"], sizes)
    s["table"], s["len"], s["refs"], s["room"] = parts[0].view(seqs, blocks), parts[1], parts[2], parts[3]
    s["k"] = _normal(g, dtype, layers, pages, cells)
    s["v"] = _normal(g, dtype, layers, pages, cells)
    s["slots"] = _ints(slots)
    s["host_slots"] = slots
    s["ko"], s["vo"] = _offsets(d)

    if kind == "pages" and case["op"] == "fork":
        s["parent"], s["child"] = _ints([slots[0]] * n), _ints(order[n:])
    if kind in ("rope", "packed"):
        cu = [0]
        for k in new:
            cu.append(cu[-1] + k)
        s["cu"], s["host_cu"] = _ints(cu), cu
        s["rows"] = max(cu[-1] + case["pad"], 1)
    if kind == "rope":
        io, rows = _TYPES[case["io"]], s["rows"]
        wide = (group + 2) * hkv * d
        s["qkv"] = _normal(g, io, rows, wide)  # one projection's rows: q, k and v
        s["q_out"] = torch.zeros(rows, group * hkv * d, device="cuda", dtype=dtype)
        f, s["scale"] = _frequencies(case)
        s["freq"] = torch.tensor(f or [0.0], dtype=torch.float64, device="cuda")
        if case["norm"]:
            s["gq"], s["gk"] = (torch.rand(d, generator=g, device="cuda") * 0.2 + 0.9 for _ in range(2))
        # position and entry of every row
        pos = [lens[i] - new[i] + j for i in range(n) for j in range(new[i])]
        s["pos"] = torch.tensor(pos, dtype=torch.int64, device="cuda")
        s["of"] = torch.tensor([slots[i] for i in range(n) for _ in range(new[i])], dtype=torch.int64, device="cuda")
    if kind in ("packed", "shared"):
        rows = s["rows"] if kind == "packed" else n
        # queries as a norm leaves them, keys of their own size
        s["q"] = _normal(g, dtype, rows, group * hkv * d)
        s["out"] = torch.zeros_like(s["q"])
    if own:
        from hymt2sharp_amd import BF16, F16, F32, PagedCache, Rope, SeqBatch
        types = {"f32": F32, "f16": F16, "bf16": BF16}
        s["cache"] = PagedCache(k=_ptr(s["k"]), v=_ptr(s["v"]), table=_ptr(s["table"]), len=_ptr(s["len"]),
                                refs=_ptr(s["refs"]), work=_ptr(s["room"]), layers=layers, pages=pages, kv_heads=hkv,
                                head_dim=d, dtype=F16 if dtype == torch.float16 else BF16, seqs=seqs, blocks=blocks)
        s["io"] = types.get(case.get("io"))
        s["batch"] = SeqBatch(slots=_ptr(s["slots"]), cu=_ptr(s["cu"]) if "cu" in s and kind != "shared" else None,
                              n=n, rows=s.get("rows", n), max_len=max(lens))
        if kind == "rope":
            s["rope"] = Rope(freq=_ptr(s["freq"]), dim=case["rot"], interleaved=case["pairs"] == "interleaved",
                             scale=s["scale"])
    torch.cuda.synchronize()
    return s


# ---- one pass: plain ---------------------------------------------------------------


def _free_pages(refs):
    return torch.argsort((refs > 0).to(torch.int32), stable=True)


def _plain_pages(s):
    c = s["case"]
    s["meta"].copy_(s["meta0"])
    table, ln, refs, k, v = s["table"], s["len"], s["refs"], s["k"], s["v"]
    if c["op"] == "compact":
        live = (refs > 0).sum()
        page = torch.arange(refs.numel(), device="cuda")
        src = page[(refs > 0) & (page >= live)]
        dst = page[(refs == 0) & (page < live)]
        to = page.clone()
        to[src] = dst
        refs[dst] = refs[src]
        refs[src] = 0
        table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    elif c["op"] == "fork":
        par, chi = s["parent"].long(), s["child"].long()
        length = ln[par].long()
        full, ends = length // PAGE, length % PAGE > 0
        fresh = _free_pages(refs)[torch.cumsum(ends, 0) - 1]
        col = torch.arange(table.shape[1], device="cuda")
        row = table[par].long()
        whole = col < full[:, None]
        refs.index_add_(0, row[whole], torch.ones_like(row[whole], dtype=torch.int32))
        src, dst = table[par, full].long()[ends], fresh[ends]
        row = torch.where(whole, row, -1)
        row[ends, full[ends]] = dst
        table[chi] = row.int()
        ln[chi] = length.int()
        refs[dst] = 1
    else:
        slot = s["slots"].long()
        length = ln[slot].long()
        more = length % PAGE == 0
        fresh = _free_pages(refs)[torch.cumsum(more, 0) - 1][more]
        table[slot[more], length[more] // PAGE] = fresh.int()
        refs[fresh] = 1
        ln[slot] = (length + 1).int()
        return [table, ln, refs]
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    return [table, ln, refs, k, v]


def _rotate(x, cos, sin, rot, interleaved):
    """x [rows][heads][d] fp32, cos and sin [rows][1][rot / 2]."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


def _plain_rope(s):
    c = s["case"]
    hkv, group, d, rot = c["hkv"], c["group"], c["d"], c["rot"]
    total = s["host_cu"][-1]
    x = s["qkv"][:total].float().view(total, (group + 2) * hkv, d)
    qk, v = x[:, :(group + 1) * hkv], x[:, (group + 1) * hkv:]
    if rot:
        angle = s["pos"].double()[:, None] * s["freq"]
        cos, sin = (f(angle).float()[:, None] * s["scale"] for f in (torch.cos, torch.sin))
        qk = _rotate(qk, cos, sin, rot, c["pairs"] == "interleaved")
    if c["norm"]:
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS)
        qk = torch.cat([qk[:, :group * hkv] * s["gq"], qk[:, group * hkv:] * s["gk"]], 1)
    s["q_out"][:total] = qk[:, :group * hkv].reshape(total, -1).to(s["q_out"].dtype)
    page = s["table"][s["of"], s["pos"] // PAGE].long()
    at = s["pos"] % PAGE
    pool_k, pool_v = s["k"][0].view(-1, hkv, PAGE * d), s["v"][0].view(-1, hkv, PAGE * d)
    head = torch.arange(hkv, device="cuda")[None, :, None]
    pool_k[page[:, None, None], head, s["ko"][at][:, None]] = qk[:, group * hkv:].to(pool_k.dtype)
    pool_v[page[:, None, None], head, s["vo"][at][:, None]] = v.to(pool_v.dtype)
    return [s["q_out"], s["k"], s["v"]]


def _gather(s, slot, length):
    """K and V of a sequence's positions, fp32 [hkv][length][d]."""
    c = s["case"]
    hkv, d = c["hkv"], c["d"]
    pages = s["table"][slot, :_blocks(length)].long()
    out = []
    for pool, off in ((s["k"], s["ko"]), (s["v"], s["vo"])):
        x = pool[0][pages].view(-1, hkv, PAGE * d)[:, :, off.reshape(-1)]
        x = x.view(-1, hkv, PAGE, d).transpose(0, 1).reshape(hkv, -1, d)
        out.append(x[:, :length].float().contiguous())
    return out


def _softmax_rows(q, k, v, limit):
    """q [hkv][m][d], k and v [hkv][len][d]; row m sees the positions below limit[m]."""
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(q.shape[-1])
    hidden = torch.arange(k.shape[1], device="cuda")[None, :] >= limit[:, None]
    scores.masked_fill_(hidden, float("-inf"))
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.matmul(scores, v) / scores.sum(-1, keepdim=True)


def _plain_attention(s):
    c = s["case"]
    hkv, group, d = c["hkv"], c["group"], c["d"]
    out = s["out"]
    for i in range(c["n"]):
        new, length = s["new"][i], s["lens"][i]
        r0 = s["host_cu"][i] if c["kind"] == "packed" else i
        if new == 0:
            continue
        k, v = _gather(s, s["host_slots"][i], length)
        for a in range(0, new, 1024):  # a part of the rows at a time
            m = min(1024, new - a)
            q = s["q"][r0 + a:r0 + a + m].float().view(m, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, m * group, d)
            limit = torch.arange(length - new + a + 1, length - new + a + m + 1, device="cuda")
            y = _softmax_rows(q, k, v, limit.repeat_interleave(group))
            out[r0 + a:r0 + a + m] = y.view(hkv, m, group, d).permute(1, 0, 2, 3).reshape(m, -1).to(out.dtype)
    return out


# ---- one pass: the framework's operators -------------------------------------------


def _ptr(t):
    return t.data_ptr()


def _calls(s):
    be, stream = _backend()
    c = s["case"]
    kind, cache = c["kind"], s["cache"]
    if kind == "pages":
        with torch.cuda.stream(stream):  # the sequences as the step before left them
            s["meta"].copy_(s["meta0"])
        if c["op"] == "extend":
            be.paged_extend(cache, _ptr(s["slots"]), c["n"])
            return [s["table"], s["len"], s["refs"]]
        if c["op"] == "fork":
            be.paged_fork(cache, _ptr(s["parent"]), _ptr(s["child"]), c["n"])
        else:
            be.paged_compact(cache)
        return [s["table"], s["len"], s["refs"], s["k"], s["v"]]
    heads = c["hkv"] * c["group"]
    if kind == "rope":
        d, e = c["d"], s["qkv"].element_size()
        wide = (c["group"] + 2) * c["hkv"] * d
        q = _ptr(s["qkv"])
        be.rope_append(cache, 0, s["batch"], q, wide, q + heads * d * e, q + (heads + c["hkv"]) * d * e, wide, s["io"],
                       heads, s["rope"], _ptr(s["gq"]) if c["norm"] else None, _ptr(s["gk"]) if c["norm"] else None,
                       EPS, _ptr(s["q_out"]))
        return [s["q_out"], s["k"], s["v"]]
    if kind == "packed":
        be.attn_packed(cache, 0, s["batch"], _ptr(s["q"]), heads, _ptr(s["out"]))
    else:
        be.attn_shared(cache, 0, s["batch"], c["prefix"], _ptr(s["q"]), heads, _ptr(s["out"]))
    return s["out"]


def run(state):
    if own:
        return _calls(state)
    kind = state["case"]["kind"]
    return {"pages": _plain_pages, "rope": _plain_rope}.get(kind, _plain_attention)(state)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    kind, n = case["kind"], case["n"]
    hkv, group, d = case["hkv"], case["group"], case["d"]
    new, lens = _lens(case)
    page = 2 * 2 * hkv * PAGE * d  # K and V of one layer
    if kind == "pages":
        ints = 4 * (case["pages"] + 4 * n)
        if case["op"] == "extend":
            return {"bytes": ints, "flops": 2 * n}
        if case["op"] == "fork":
            copies = sum(k % PAGE > 0 for k in lens)
            ints += 4 * (n + 1) * _blocks(lens[0])
        else:
            live = _pages_of(case)
            copies = min(case["moved"], live, case["pages"] - live)
            ints += 8 * live
        return {"bytes": ints + 2 * copies * page * case["layers"], "flops": 2 * n}
    if kind == "rope":
        rows, e = sum(new), 4 if case["io"] == "f32" else 2
        return {"bytes": rows * (group + 2) * hkv * d * (e + 2), "flops": 10 * rows * (group + 1) * hkv * d}
    rows = sum(new)
    seen = sum(k * (x - k) + k * (k + 1) // 2 for k, x in zip(new, lens))
    held = sum(x for k, x in zip(new, lens) if k) - (n - 1) * case.get("prefix", 0)
    return {"bytes": 2 * held * hkv * d * 2 + 2 * rows * group * hkv * d * 2, "flops": 4 * d * group * hkv * seen}


# ---- the same in 64 bits -----------------------------------------------------------


def _exact_pages(s):
    c = s["case"]
    table, held, refs = (s[x].cpu().numpy().copy() for x in ("table", "len", "refs"))
    pairs = []
    if c["op"] == "extend":
        for slot in s["host_slots"]:
            if held[slot] % PAGE == 0:
                p = int(np.flatnonzero(refs == 0)[0])
                table[slot, held[slot] // PAGE], refs[p] = p, 1
            held[slot] += 1
    elif c["op"] == "fork":
        for a, b in zip(s["parent"].tolist(), s["child"].tolist()):
            for j in range(_blocks(int(held[a]))):
                p = int(table[a, j])
                if (j + 1) * PAGE > held[a]:
                    q = int(np.flatnonzero(refs == 0)[0])
                    pairs.append((p, q))
                    p = q
                table[b, j] = p
                refs[p] += 1
            held[b] = held[a]
    else:
        live = int((refs > 0).sum())
        holes = [p for p in range(live) if refs[p] == 0]
        movers = [p for p in range(live, len(refs)) if refs[p] > 0]
        for p, q in zip(movers, holes):
            table[table == p] = q
            refs[q], refs[p] = refs[p], 0
            pairs.append((p, q))
    ints = [torch.from_numpy(x).cuda() for x in (table, held, refs)]
    if c["op"] == "extend":
        return ints
    pools = []
    for x in (s["k"], s["v"]):
        x = x.clone()
        for p, q in pairs:
            x[:, q] = x[:, p]
        pools.append(x)
    return ints + pools


def _exact_rope(s):
    c = s["case"]
    hkv, group, d, rot = c["hkv"], c["group"], c["d"], c["rot"]
    heads, total = hkv * group, s["host_cu"][-1]
    x = s["qkv"][:total].double().view(total, -1, d)
    y = x.clone()
    if rot:
        turn = torch.polar(torch.full((total, rot // 2), s["scale"], dtype=torch.float64, device="cuda"),
                           s["pos"].double().unsqueeze(1) * s["freq"]).unsqueeze(1)
        i = torch.arange(rot // 2, device="cuda")
        first, second = (2 * i, 2 * i + 1) if c["pairs"] == "interleaved" else (i, i + rot // 2)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
    if c["norm"]:
        y = y / (y.square().sum(-1, keepdim=True) / d + EPS).sqrt()
        y[:, :heads] *= s["gq"].double()
        y[:, heads:] *= s["gk"].double()
    q = s["q_out"].double()
    q[:total] = y[:, :heads].reshape(total, -1)
    k = s["k"].double().view(-1, hkv, PAGE * d)
    v = s["v"].double().view(-1, hkv, PAGE * d)
    dims = torch.arange(d, device="cuda")
    r = 0
    for i, slot in enumerate(s["host_slots"]):
        start = s["lens"][i] - s["new"][i]
        for p0 in range(start, s["lens"][i]):
            if p0 % PAGE and p0 > start:
                continue  # the rows of a page are written together
            m = min(PAGE - p0 % PAGE, s["lens"][i] - p0)
            page = int(s["table"][slot, p0 // PAGE])
            t = torch.arange(p0 % PAGE, p0 % PAGE + m, device="cuda")[:, None]
            at_k = (t // 16) * 16 * d + (dims // 8) * 128 + (t % 16) * 8 + dims % 8
            at_v = (t // 32) * 32 * d + (t % 16 // 4) * 8 * d + dims * 8 + (t % 32 // 16) * 4 + t % 4
            for h in range(hkv):
                k[page, h, at_k] = y[r:r + m, heads + h]
                v[page, h, at_v] = x[r:r + m, heads + hkv + h]
            r += m
    return [q, k.view(s["k"].shape), v.view(s["v"].shape)]


def _exact_attention(s):
    c = s["case"]
    hkv, group, d = c["hkv"], c["group"], c["d"]
    out = s["out"].double()
    row = 0
    for i, slot in enumerate(s["host_slots"]):
        new, length = s["new"][i], s["lens"][i]
        pages = s["table"][slot, :_blocks(length)].long()
        for h in range(hkv):
            if not new:
                break
            cut = slice(h * PAGE * d, (h + 1) * PAGE * d)
            k = s["k"][0, pages, cut].double().view(-1, 4, d // 8, 16, 8).permute(0, 1, 3, 2, 4).reshape(-1, d)[:length]
            v = s["v"][0, pages, cut].double().view(-1, 2, 4, d, 2, 4).permute(0, 1, 4, 2, 5, 3).reshape(-1, d)[:length]
            kt = k.t().contiguous()
            for g in range(group):
                col = slice((h * group + g) * d, (h * group + g + 1) * d)
                for a in range(0, new, 2048):
                    m = min(2048, new - a)
                    w = torch.mm(s["q"][row + a:row + a + m, col].double(), kt).mul_(d ** -0.5)
                    last = length - new + a
                    w += torch.full_like(w, float("-inf")).triu_(last + 1)
                    out[row + a:row + a + m, col] = torch.mm(torch.softmax(w, -1), v)
        row += new
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pages":
        return _exact_pages(s)
    return _exact_rope(s) if kind == "rope" else _exact_attention(s)
