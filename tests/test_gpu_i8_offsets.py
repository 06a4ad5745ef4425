"""The 8-bit integer operators where an element lies more than 2^32 elements from
its tensor's first: outputs whose rows are far apart, tokens and channels of long
rows of codes, and many rows of values.  Only the parts that are compared hold
inputs; the rest is whatever the allocation held.  The bounds are those of the
operators' own tests."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.i8_cases import U32, bf16_bits, bf16_val, codes, codes_of, norm_rows, product, scales
from tests.test_gpu_i8_gemm import TILES, check, check_glu

pytestmark = pytest.mark.gpu

FAR = 1 << 32


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


class Memory:
    """Allocations of one test; the test is skipped where one finds no room."""

    def __init__(self, be):
        self.be, self.ptrs = be, []

    def alloc(self, nbytes):
        try:
            self.ptrs.append(self.be.alloc(nbytes))
        except MemoryError:
            self.close()
            pytest.skip(f"no room for {nbytes} bytes")
        return self.ptrs[-1]

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.alloc(a.nbytes)
        self.be.upload(p, a)
        return p

    def close(self):
        for p in self.ptrs:
            self.be.free(p)
        self.ptrs = []


@pytest.fixture
def mem(be):
    m = Memory(be)
    yield m
    m.close()


@pytest.mark.parametrize("out", ["f32", "acc", "bf16", "glu"])
@pytest.mark.parametrize("ldy", [(1 << 27) + 8, (1 << 27) + 9])
def test_output_rows_far_apart(be, mem, monkeypatch, out, ldy):
    """Rows ldy apart, the last more than 2^32 elements from the first; whole
    16-byte stores (ldy a multiple of 8) and single elements.  The values on
    either side of each row stay as they were."""
    m, n, k, pad = 40, 200, 256, 16
    assert (m - 1) * ldy > FAR
    half = out in ("bf16", "glu")
    w, x, up = codes(1, n, k), codes(2, m, k), codes(3, n, k)
    ws, us, xs = scales(4, n), scales(5, n), scales(6, m, 1e-3, 1e-1)
    y0 = np.random.default_rng(7).standard_normal((m, n)).astype(np.float32)
    before = np.full((m, n + 2 * pad), 0x7B7B if half else 123.0, np.uint16 if half else np.float32)
    if out == "acc":
        before[:, pad:-pad] = y0
    es = before.itemsize
    dw, dws, dx, dxs, du, dus = (mem.put(a) for a in (w, ws, x, xs, up, us))
    y = mem.alloc(((m - 1) * ldy + n + 2 * pad) * es) + pad * es
    at = [y + (t * ldy - pad) * es for t in range(m)]
    for tile in TILES:
        monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
        for p, row in zip(at, before):
            be.upload(p, row)
        if out == "glu":
            be.gemm_i8_swiglu(dw, dws, du, dus, n, k, dx, dxs, m, y, ld=ldy)
        else:
            be.gemm_i8(dw, dws, n, k, dx, dxs, m, y, ldy=ldy, accumulate=out == "acc", out_bf16=out == "bf16")
        got = np.stack([be.download(np.empty_like(before[0]), p) for p in at])
        assert (got[:, :pad] == before[:, :pad]).all() and (got[:, -pad:] == before[:, -pad:]).all(), tile
        got = got[:, pad:-pad]
        if out == "glu":
            check_glu(got, w, ws, up, us, x, xs)
        else:
            check(got, product(w, ws, x, xs), out, y0)


@pytest.mark.parametrize("tile", ["16x16", "64x32", "64x64", "96x64", "128x128", "256x256"])
def test_tokens_past_32_bits(be, mem, monkeypatch, tile):
    """The last tokens of more than 2^32 codes."""
    k, m, n, tail = 65536, FAR // 65536 + 77, 36, 300
    w, x, up = codes(1, n, k), codes(2, tail, k), codes(3, n, k)
    ws, us, xs = scales(4, n, 1e-6, 1e-4), scales(5, n, 1e-6, 1e-4), scales(6, tail, 1e-3, 1e-1)
    dw, dws, du, dus = (mem.put(a) for a in (w, ws, up, us))
    dx, dxs, y = mem.alloc(m * k), mem.alloc(4 * m), mem.alloc(4 * m * n)
    be.upload(dx + (m - tail) * k, x)
    be.upload(dxs + 4 * (m - tail), xs)
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    be.gemm_i8(dw, dws, n, k, dx, dxs, m, y)
    check(be.download(np.empty((tail, n), np.float32), y + 4 * (m - tail) * n), product(w, ws, x, xs), "f32")
    be.gemm_i8_swiglu(dw, dws, du, dus, n, k, dx, dxs, m, y)
    check_glu(be.download(np.empty((tail, n), np.uint16), y + 2 * (m - tail) * n), w, ws, up, us, x, xs)


@pytest.mark.parametrize("tile", ["16x16", "64x16", "64x32", "64x64", "96x64", "128x128", "256x256"])
@pytest.mark.parametrize("m", [3, 40])
def test_channels_past_32_bits(be, mem, monkeypatch, tile, m):
    """The last channels of more than 2^32 codes, of gate and up alike."""
    k, n, tail = 65536, FAR // 65536 + 77, 300
    w, x, up = codes(1, tail, k), codes(2, m, k), codes(3, tail, k)
    ws, us, xs = scales(4, tail, 1e-6, 1e-4), scales(5, tail, 1e-6, 1e-4), scales(6, m, 1e-3, 1e-1)
    dx, dxs, y = mem.put(x), mem.put(xs), mem.alloc(4 * m * n)
    dw, dws, du, dus = mem.alloc(n * k), mem.alloc(4 * n), mem.alloc(n * k), mem.alloc(4 * n)
    for q, s, c, v in ((dw, dws, w, ws), (du, dus, up, us)):
        be.upload(q + (n - tail) * k, c)
        be.upload(s + 4 * (n - tail), v)
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    be.gemm_i8(dw, dws, n, k, dx, dxs, m, y, out_bf16=True)
    got = be.download(np.empty((m, n), np.uint16), y)[:, n - tail:]
    check(got, product(w, ws, x, xs), "bf16")
    be.gemm_i8_swiglu(dw, dws, du, dus, n, k, dx, dxs, m, y)
    got = be.download(np.empty((m, n), np.uint16), y)[:, n - tail:]
    check_glu(got, w, ws, up, us, x, xs)


def test_rows_past_32_bits(be, mem):
    """The last rows of more than 2^32 values: codes of fp32 and of bf16 rows,
    and the norm after an addition."""
    n, tail = 8192, 5
    m = FAR // n + 11
    rng = np.random.default_rng(1)
    x = rng.standard_normal((tail, n)).astype(np.float32)
    d = bf16_bits(rng.standard_normal((tail, n)))
    g = rng.uniform(0.8, 1.2, n).astype(np.float32)
    dg, dx, dd, dq, ds = mem.put(g), mem.alloc(4 * m * n), mem.alloc(2 * m * n), mem.alloc(m * n), mem.alloc(4 * m)
    t = m - tail
    be.upload(dx + 4 * t * n, x)
    be.upload(dd + 2 * t * n, d)

    def got():
        return (be.download(np.empty((tail, n), np.int8), dq + t * n),
                be.download(np.empty(tail, np.float32), ds + 4 * t))

    for p, dtype, v in ((dx, N.F32, x), (dd, N.BF16, bf16_val(d))):
        be.to_i8(p, m, n, dq, ds, x_dtype=dtype)
        q, a = codes_of(v)
        got_q, got_s = got()
        np.testing.assert_array_equal(got_q, q)
        np.testing.assert_array_equal(got_s, (a / 127.0).astype(np.float32))
    be.rows_rmsnorm_i8(dx, m, n, dg, 1e-5, dq, ds, add=dd)
    h, q, s = norm_rows(x, bf16_val(d), g, 1e-5)
    got_q, got_s = got()
    np.testing.assert_array_equal(be.download(np.empty((tail, n), np.float32), dx + 4 * t * n), h)
    np.testing.assert_array_equal(got_q, q)
    assert (np.abs(got_s - s) <= U32 * (1 + 2.0 ** -10) * s).all()
