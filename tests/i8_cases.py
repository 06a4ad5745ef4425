"""Inputs and plain references of the 8-bit integer operators
(hymt_to_i8, hymt_rows_rmsnorm_i8, hymt_gemm_i8, hymt_gemm_i8_swiglu)."""
import numpy as np

from hymt2sharp_amd import synth as S

U32 = 2.0 ** -24  # half a step of fp32, relative
U16 = 2.0 ** -8   # half a step of bf16, relative


def bf16_bits(a):
    return S.f32_to_bf16_bits(np.ascontiguousarray(a, dtype=np.float32)).reshape(np.shape(a))


def bf16_val(b):
    return S.bf16_bits_to_f32(np.ascontiguousarray(b)).reshape(np.shape(b))


def codes_of(v):
    """Codes and max|v| of rows of fp64 values: rint(127 v / a), ties to even
    (127 v is exact for values of 46 bits, and the quotient correctly rounded)."""
    v = np.asarray(v, np.float64)
    ok = np.isfinite(v).all(1)
    a = np.where(ok, np.abs(np.where(np.isfinite(v), v, 0)).max(1), np.nan)
    q = np.zeros(v.shape, np.int8)
    some = ok & (a > 0)
    q[some] = np.rint(127.0 * v[some] / a[some, None]).astype(np.int8)
    return q, a


def norm_rows(x, add, w, eps):
    """(x after the addition, codes, fp64 scales) of rows_rmsnorm_i8."""
    with np.errstate(invalid="ignore", over="ignore"):
        h = x if add is None else (x + add).astype(np.float32)
        d = h.astype(np.float64)
        q, a = codes_of(d * w.astype(np.float64))
        root = np.sqrt((d * d).mean(1) + float(np.float32(eps)))
        s = np.where(a == 0, 0.0, a / 127.0 / np.where(a == 0, 1.0, root))
    return h, q, s


def product(w, ws, x, xs):
    """fp64 y[m][n]: the int8 sums are exact in fp64 (below 2^53)."""
    return (x.astype(np.float64) @ w.astype(np.float64).T) * ws.astype(np.float64) * xs.astype(np.float64)[:, None]


def codes(seed, rows, k, extreme=False):
    rng = np.random.default_rng(seed)
    if extreme:
        return rng.choice(np.array([-128, 127], np.int8), (rows, k))
    return rng.integers(-127, 128, (rows, k), dtype=np.int8)


def scales(seed, n, lo=1e-4, hi=1e-2):
    return np.exp(np.random.default_rng(seed).uniform(np.log(lo), np.log(hi), n)).astype(np.float32)


class Room:
    """Device buffers of one test, each between 256 guard bytes of 0xA5."""

    G = 256

    def __init__(self, be):
        self.be, self.bufs = be, []

    def put(self, a, offset=0):
        """`a` on the device, `offset` bytes past a 256-byte boundary."""
        a = np.ascontiguousarray(a)
        raw = np.full(2 * self.G + offset + a.nbytes, 0xA5, np.uint8)
        raw[self.G + offset:self.G + offset + a.nbytes] = a.reshape(-1).view(np.uint8)
        p = self.be.alloc(raw.nbytes)
        self.be.upload(p, raw)
        self.bufs.append((p, raw.nbytes, self.G + offset, a.nbytes))
        return p + self.G + offset

    def get(self, ptr, like):
        out = np.empty_like(np.ascontiguousarray(like))
        return self.be.download(out, ptr)

    def close(self):
        """Checks every guard byte and frees the buffers."""
        bad = []
        for p, total, at, n in self.bufs:
            raw = self.be.download(np.empty(total, np.uint8), p)
            if (raw[:at] != 0xA5).any() or (raw[at + n:] != 0xA5).any():
                bad.append((hex(p), n))
            self.be.free(p)
        self.bufs = []
        assert not bad, f"bytes outside a buffer were written: {bad}"
