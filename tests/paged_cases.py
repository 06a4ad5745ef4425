"""Inputs and plain references of the multi-sequence cache's operators
(hymt_paged_*, hymt_rope_append, hymt_attn_packed, hymt_attn_shared): numpy, in 64
bits, from the definitions in include/hymt_hip.h."""
import numpy as np

from hymt2sharp_amd import _native as N
from tests.i8_cases import Room, bf16_bits, bf16_val

PAGE = 64
# half a step of the type, relative, and of its subnormal numbers
U = {N.F16: 2.0 ** -11, N.BF16: 2.0 ** -8}
TINY = {N.F16: 2.0 ** -25, N.BF16: 2.0 ** -134}
U32 = 2.0 ** -24


def to_bits(a, dt):
    a = np.ascontiguousarray(a, np.float32)
    if dt == N.BF16:
        return np.where(np.isnan(a), np.uint16(0x7FC0), bf16_bits(a)).astype(np.uint16)
    with np.errstate(over="ignore"):
        return a.astype(np.float16).view(np.uint16)


def from_bits(b, dt):
    b = np.ascontiguousarray(b, np.uint16)
    return bf16_val(b) if dt == N.BF16 else b.view(np.float16).astype(np.float32)


def offsets(d):
    t, i = np.arange(PAGE)[:, None], np.arange(d)[None, :]
    ko = ((t // 16 * (d // 8) + i // 8) * 16 + t % 16) * 8 + i % 8
    vo = ((4 * (t // 32) + t // 4 % 4) * d + i) * 8 + 4 * (t // 16 % 2) + t % 4
    return ko, vo


def blocks_of(n):
    return -(-n // PAGE)


class Cache:
    """A multi-sequence cache in host memory: pools of bits that every position
    not set is garbage in (NaN among it), table, lengths, references, work."""

    def __init__(self, seed, layers=1, pages=8, kv_heads=2, d=128, dt=N.BF16, seqs=4, blocks=6):
        self.rng = np.random.default_rng(seed)
        self.layers, self.pages, self.kv_heads, self.d, self.dt = layers, pages, kv_heads, d, dt
        self.seqs, self.blocks = seqs, blocks
        shape = (layers, pages, kv_heads, PAGE * d)
        self.k, self.v = (self.rng.integers(0, 1 << 16, shape, dtype=np.uint16) for _ in range(2))
        self.table = np.full((seqs, blocks), -1, np.int32)
        self.len = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.work = np.zeros(N.paged_work(pages), np.int32)
        self.ko, self.vo = offsets(d)

    def give(self, slot, length, pages=None, values=True):
        """The slot gets `length` positions in any free pages, filled with normal
        values (garbage past them)."""
        free = [int(p) for p in np.flatnonzero(self.refs == 0)]
        self.rng.shuffle(free)
        for b in range(blocks_of(length)):
            p = free.pop() if pages is None else pages[b]
            self.table[slot, b] = p
            self.refs[p] += 1
            if values:
                n = min(PAGE, length - b * PAGE)
                for pool, off in ((self.k, self.ko), (self.v, self.vo)):
                    x = self.rng.standard_normal((self.layers, self.kv_heads, n, self.d))
                    pool[:, p][:, :, off[:n]] = to_bits(x, self.dt)
        self.len[slot] = length

    def rows(self, layer, slot, length):
        """K and V [kv_heads][length][d] as fp64."""
        out = []
        for pool, off in ((self.k, self.ko), (self.v, self.vo)):
            x = np.zeros((self.kv_heads, blocks_of(length) * PAGE, self.d))
            for b in range(blocks_of(length)):
                x[:, b * PAGE:(b + 1) * PAGE] = from_bits(pool[layer, self.table[slot, b]][:, off], self.dt)
            out.append(x[:, :length])
        return out

    # ---- on the device
    def put(self, room):
        c = N.PagedCache(layers=self.layers, pages=self.pages, kv_heads=self.kv_heads, head_dim=self.d, dtype=self.dt,
                         seqs=self.seqs, blocks=self.blocks)
        for name in ("k", "v", "table", "len", "refs", "work"):
            setattr(c, name, room.put(getattr(self, name)))
        return c

    def get(self, room, c, *names):
        return [room.get(getattr(c, n), getattr(self, n)) for n in names]


def batch(room, slots, cu=None, rows=None, max_len=0):
    b = N.SeqBatch(slots=room.put(np.asarray(slots, np.int32)), n=len(slots), max_len=max_len)
    if cu is not None:
        b.cu = room.put(np.asarray(cu, np.int32))
    b.rows = rows if rows is not None else (cu[-1] if cu is not None else len(slots))
    return b


# ---- attention ---------------------------------------------------------------------


def attend(q, k, v, limit, scale, dt, out_dt=None):
    """(out, tolerance) of one kv head: q [m][d], k and v [len][d], row i sees the
    positions below limit[i].

    The tolerance, A = sum p |v| being the weights' mean of |v|: the weights are rounded
    to the type (relative u each, and the kernel may divide by the sum before or
    after: 2 u A; in fp16 a weight that is subnormal is off by 2^-25 of the
    largest, which is 1: n 2^-25 max |v|); a score is a sum of d products in
    fp32, relative (d + 8) 2^-24 of sum |q k| (and as much again for the largest
    it is compared with), the exponential and its argument 2^-20 of |s|; the sums over n positions
    2 n 2^-24 A; splitting and joining parts a few more fp32 roundings; the
    result is rounded once, u' |out|."""
    out_dt = dt if out_dt is None else out_dt
    m, d = q.shape
    out, tol = np.zeros((m, d)), np.zeros((m, d))
    # an infinity or a NaN that a row sees makes its result one: no tolerance there
    ka, va = (np.abs(np.where(np.isfinite(x), x, 0)) for x in (k, v))
    for i in range(m):
        n = int(limit[i])
        if n <= 0:
            continue
        s = k[:n] @ q[i] * scale
        w = np.exp(s - s.max())
        p = w / w.sum()
        out[i] = p @ v[:n]
        a = p @ va[:n]
        size = (ka[:n] @ np.abs(q[i])).max() * abs(scale)
        rel = 2 * U[dt] + 2 * (d + 8) * U32 * size + 2.0 ** -20 * (size + 1) + (2 * n + 64) * U32
        tol[i] = a * rel + (n * 2.0 ** -25 * va[:n].max() if dt == N.F16 else 0) + U[out_dt] * np.abs(out[i])
        tol[i] += TINY[out_dt]
    return out, tol


def attention(cache, layer, slots, cu, q, heads, scale=None, prefix=0, out_dt=None):
    """(out [rows][heads * d], tolerance, written rows) in 64 bits."""
    d, hkv = cache.d, cache.kv_heads
    g = heads // hkv
    scale = d ** -0.5 if scale is None else float(np.float32(scale))
    out, tol = np.zeros((q.shape[0], heads * d)), np.zeros((q.shape[0], heads * d))
    done = np.zeros(q.shape[0], bool)
    common = min(prefix, int(cache.len[slots[0]]) // PAGE * PAGE) if len(slots) else 0
    for e, slot in enumerate(slots):
        a, b = (e, e + 1) if cu is None else (cu[e], cu[e + 1])
        if a == b:
            continue
        done[a:b] = True
        n = int(cache.len[slot])
        k, v = cache.rows(layer, slot, n)
        if common and n:
            kp, vp = cache.rows(layer, slots[0], min(common, n))
            k[:, :common], v[:, :common] = kp, vp
        limit = n - (b - a) + 1 + np.arange(b - a)
        for h in range(heads):
            c = slice(h * d, (h + 1) * d)
            out[a:b, c], tol[a:b, c] = attend(q[a:b, c].astype(np.float64), k[h // g], v[h // g], limit, scale, cache.dt,
                                              out_dt)
    return out, tol, done


def check_rows(got_bits, want, tol, done, before_bits, dt):
    """Rows of the batch within their tolerance, all others as they were."""
    got = from_bits(got_bits, dt).astype(np.float64)
    np.testing.assert_array_equal(got_bits[~done], before_bits[~done])
    nan = np.isnan(want)
    assert (np.isnan(got)[done] == nan[done]).all()
    inf = np.isinf(want)
    assert (got[inf & done[:, None]] == want[inf & done[:, None]]).all()
    ok = done[:, None] & ~nan & ~inf
    with np.errstate(invalid="ignore"):
        bad = ok & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           float(np.max(np.where(ok, np.abs(got - want) / np.maximum(tol, 1e-300), 0))))


# ---- rotary append -----------------------------------------------------------------


def rotated(x, pos, freq, scale, dim, interleaved, w, eps):
    """(y, tolerance without the last rounding) of rows x [rows][heads][d].

    cosine and sine are off by 2^-22 each at most (the angle's fraction rounded to fp32
    and the functions' own error), a rotated value is two products and a sum of
    such: (|x0| + |x1|) |scale| 2^-21; the norm's sum of d squares, its root
    and the products (d + 16) 2^-24 relative, and the rotation's error goes into it as
    into the value itself."""
    x = x.astype(np.float64)
    d = x.shape[-1]
    y, err = x.copy(), np.zeros_like(x)
    if dim:
        half = dim // 2
        ang = pos[:, None].astype(np.float64) * freq
        c, s = np.cos(ang)[:, None] * scale, np.sin(ang)[:, None] * scale
        i = np.arange(half)
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[..., p] = x[..., p] * c - x[..., q] * s
        y[..., q] = x[..., q] * c + x[..., p] * s
        err[..., p] = err[..., q] = (np.abs(x[..., p]) + np.abs(x[..., q])) * abs(scale) * 2.0 ** -21
    if w is not None:
        root = 1 / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps)))
        rel = (np.abs(y) * err).sum(-1, keepdims=True) / np.maximum((y * y).sum(-1, keepdims=True), 1e-300)
        y = y * root * w
        err = err * root * np.abs(w) + np.abs(y) * ((d + 16) * U32 + rel)
    return y, err + np.abs(y) * 2 * U32
