"""hymt_gemm_i8 and hymt_gemm_i8_swiglu on the GPU against fp64 products of the
same codes and scales.

Bounds, u = 2^-24 (half a step of fp32): the int32 sum is exact, its
conversion to fp32 and the two products with the scales round once each, so an
fp32 result is within 3 u (1 + 2 u) of y, taken as 3.01 u |y|.  Accumulating fuses the
last product with the addition: 2.01 u |v| + u |y0 + v|.  bf16 rounds once more:
2^-8 |y| (1 + 2^-10).  SwiGLU: g and u are within 3.01 u; the exponential's argument is
off by the 3.01 u of g, a product's rounding and its constant's, 5 u |g| in
all, relative on e^-g, the hardware's exponential, reciprocal and the two
products add 8 u, and u's own 3.01: (5 |g| + 16) u relative in fp32, then bf16's
rounding.  Below fp32's normal range results flush or round, 2^-125 absolute; so
does the reciprocal 1 / (1 + e^-g), which is below 2^-126 from g = -87.3 on and is
then 0 in place of a value below 2^-126: |g u| 2^-126 in the result.

Whatever kernel a shape takes, the bits of a row are the same."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from tests.i8_cases import U16, U32, Room, bf16_val, codes, product, scales

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -125
# tokens, channels, k: one token, one channel, odd and ragged sizes, tile
# borders on either side, the model's own, the largest k
SHAPES = [(1, 1, 256), (1, 17, 384), (2, 64, 256), (3, 130, 640), (16, 16, 2048), (17, 33, 1152), (1, 2048, 2048),
          (61, 2048, 6144), (64, 100, 2048), (65, 257, 896), (127, 129, 512), (128, 128, 256), (129, 191, 384),
          (200, 1000, 2048), (256, 512, 768), (300, 515, 2048), (700, 2048, 2048), (513, 6145, 256),
          (1, 20001, 2048), (33, 9999, 512), (2, 40, 65536), (2049, 130, 384)]
GLU = [(1, 1, 256), (1, 6144, 2048), (3, 65, 384), (16, 128, 256), (61, 6144, 2048), (65, 63, 640), (130, 100, 512),
       (300, 515, 2048), (700, 1000, 1152), (513, 3001, 256)]


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def run(be, w, ws, x, xs, out, ldy=None, offset=0, y0=None, up=None, us=None, ms=None):
    """y of one call (of a call per part of the rows with ms) into rows ldy
    apart; what lies between and around the rows stays as it was."""
    n, k = w.shape
    m = x.shape[0]
    ldy = ldy or n
    half = out in ("bf16", "glu")
    buf = np.full((m, ldy), 0x7B7B if half else 123.0, np.uint16 if half else np.float32)
    if y0 is not None:
        buf[:, :n] = y0
    r = Room(be)
    dw, dws, dx, dxs = r.put(w), r.put(ws), r.put(x), r.put(xs)
    dy = r.put(buf, offset)
    if out == "glu":
        du, dus = r.put(up), r.put(us)
    t = 0
    for p in ms or [m]:
        a = (dx + t * k, dxs + 4 * t, p, dy + t * ldy * buf.itemsize)
        if out == "glu":
            be.gemm_i8_swiglu(dw, dws, du, dus, n, k, *a, ld=ldy)
        else:
            be.gemm_i8(dw, dws, n, k, *a, ldy=ldy, accumulate=out == "acc", out_bf16=out == "bf16")
        t += p
    got = r.get(dy, buf)
    r.close()
    assert (got[:, n:] == buf[:, n:]).all()
    return got[:, :n]


def check(got, y, out, y0=None):
    if out == "acc":
        v, y = y, y0.astype(np.float64) + y
        tol = 2.01 * U32 * np.abs(v) + U32 * np.abs(y)
    else:
        tol = 3.01 * U32 * np.abs(y)
    if out == "bf16":
        got, tol = bf16_val(got), np.abs(y) * (U16 * (1 + 2.0 ** -10))
    assert (np.abs(got.astype(np.float64) - y) <= tol + TINY).all()


def check_glu(got, w, ws, up, us, x, xs):
    g, u = product(w, ws, x, xs), product(up, us, x, xs)
    with np.errstate(over="ignore"):
        y = g / (1 + np.exp(-g)) * u
    tol = np.abs(y) * (U16 + (5 * np.abs(g) + 16) * U32) * (1 + 2.0 ** -7)
    tol += np.abs(g * u) * 2.0 ** -126
    assert (np.abs(bf16_val(got).astype(np.float64) - y) <= tol + TINY).all()


@pytest.mark.parametrize("out", ["f32", "acc", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_i8(be, m, n, k, out):
    w, x = codes(n + k, n, k), codes(m + k, m, k)
    ws, xs = scales(n, n), scales(m, m, 1e-3, 1.0)
    y0 = np.random.default_rng(5).standard_normal((m, n)).astype(np.float32) if out == "acc" else None
    check(run(be, w, ws, x, xs, out, y0=y0), product(w, ws, x, xs), out, y0)


@pytest.mark.parametrize("m,f,k", GLU)
def test_gemm_i8_swiglu(be, m, f, k):
    w, up, x = codes(f + k, f, k), codes(f + k + 1, f, k), codes(m + k, m, k)
    ws, us, xs = scales(f, f, 1e-5, 1e-3), scales(f + 1, f, 1e-5, 1e-3), scales(m, m, 1e-2, 1.0)
    check_glu(run(be, w, ws, x, xs, "glu", up=up, us=us), w, ws, up, us, x, xs)


@pytest.mark.parametrize("m,n,k", [(1, 70, 8192), (100, 70, 8192), (3, 20, 65536), (300, 300, 2048)])
def test_largest_sums(be, m, n, k):
    """Codes of -128 and 127 alone, and rows of -128 throughout: sums up to 2^30."""
    w, x = codes(1, n, k, extreme=True), codes(2, m, k, extreme=True)
    w[0], x[0] = -128, -128
    one = np.ones(n, np.float32), np.ones(m, np.float32)
    y = run(be, w, one[0], x, one[1], "f32")
    assert y[0, 0] == 128.0 * 128.0 * k
    check(y, product(w, one[0], x, one[1]), "f32")


@pytest.mark.parametrize("out", ["f32", "acc", "bf16", "glu"])
@pytest.mark.parametrize("ldy,offset", [(72, 0), (75, 4), (70, 2), (128, 8)])
def test_rows_apart_and_off_alignment(be, out, ldy, offset):
    """A column range of a wider matrix, rows at odd offsets."""
    if out in ("f32", "acc") and offset % 4:
        offset = 4
    for m in (1, 40, 150):
        n, k = 70, 512
        w, x, up = codes(1, n, k), codes(2, m, k), codes(3, n, k)
        ws, us, xs = scales(4, n), scales(5, n), scales(6, m, 1e-3, 1e-1)
        y0 = np.random.default_rng(7).standard_normal((m, n)).astype(np.float32) if out == "acc" else None
        got = run(be, w, ws, x, xs, out, ldy, offset, y0, up, us)
        if out == "glu":
            check_glu(got, w, ws, up, us, x, xs)
        else:
            check(got, product(w, ws, x, xs), out, y0)


@pytest.mark.parametrize("out", ["f32", "acc", "bf16", "glu"])
@pytest.mark.parametrize("n,k", [(2048, 2048), (6144, 2048), (2048, 6144), (515, 640)])
def test_a_row_has_the_same_bits_in_every_call(be, out, n, k):
    """The rows of a long call against calls of their own and of other lengths,
    which take other kernels."""
    m = 700
    w, x, up = codes(1, n, k), codes(2, m, k), codes(3, n, k)
    ws, us, xs = scales(4, n), scales(5, n), scales(6, m, 1e-3, 1e-1)
    y0 = np.random.default_rng(7).standard_normal((m, n)).astype(np.float32) if out == "acc" else None
    a = run(be, w, ws, x, xs, out, None, 0, y0, up, us)
    for ms in ([1, 1, 2, 3, 12, 45, 64, 90, 111, 128, 243], [16, 32, 61, 191, 400], [333, 367]):
        assert sum(ms) == m
        b = run(be, w, ws, x, xs, out, None, 0, y0, up, us, ms)
        np.testing.assert_array_equal(a, b)


def test_nan_and_zero_scales_stay_in_their_rows(be):
    """A token's NaN scale (a row with a NaN before the quantiser), also one of
    all ones, makes its outputs NaN and no others; zero codes or scales give
    zeros."""
    n, k = 300, 512
    for m, bits in ((3, 0x7FC00000), (90, 0xFFFFFFFF), (3, 0x7FFFFFFF)):
        w, x = codes(1, n, k), codes(2, m, k)
        ws, xs = scales(3, n), scales(4, m)
        x[1] = 0
        xs.view(np.uint32)[1] = bits
        xs[2] = 0
        ws[7] = 0
        for out in ("f32", "bf16", "glu"):
            got = run(be, w, ws, x, xs, out, up=w, us=ws)
            got = got if out == "f32" else bf16_val(got)
            assert np.isnan(got[1]).all()
            rest = np.delete(got, 1, 0)
            assert np.isfinite(rest).all() and not rest[:, 7].any() and not got[2].any()


def test_no_tokens(be):
    r = Room(be)
    p = r.put(np.full(4096, 3, np.int8))
    be.gemm_i8(p, p, 4, 256, p, p, 0, p)
    be.gemm_i8_swiglu(p, p, p, p, 4, 256, p, p, 0, p)
    assert (r.get(p, np.empty(4096, np.int8)) == 3).all()
    r.close()


def test_offsets_past_32_bits(be):
    """Rows of an output and of codes that lie more than 2^31 elements (and
    2^32 bytes) from the first: the last tokens of a long, wide product."""
    n, k, m = 130, 256, 8_500_000  # x: 2.2 GB of codes, y 4.4 GB
    try:
        dx = be.alloc(m * k)
        dy = be.alloc(4 * m * n)
    except MemoryError:
        pytest.skip("no room for matrices of 2.2 and 4.4 GB")
    r = Room(be)
    try:
        w, ws = codes(1, n, k), scales(2, n)
        tail = 300
        x = codes(3, tail, k)
        xs = scales(4, tail)
        ds = be.alloc(4 * m)
        be.upload(dx + (m - tail) * k, x)
        be.upload(ds + 4 * (m - tail), xs)
        dw, dws = r.put(w), r.put(ws)
        be.gemm_i8(dw, dws, n, k, dx, ds, m, dy)
        got = be.download(np.empty((tail, n), np.float32), dy + 4 * (m - tail) * n)
        be.free(ds)
        check(got, product(w, ws, x, xs), "f32")
    finally:
        be.free(dx)
        be.free(dy)
        r.close()


TILES = ["16x16", "32x16", "48x16", "64x16", "32x32", "64x32", "64x64", "96x64", "128x64", "128x96", "128x128",
         "192x128", "256x128", "192x256", "256x256"]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 256), (2, 190, 384), (31, 257, 640), (130, 100, 1152), (300, 520, 2048)])
def test_every_tile(be, monkeypatch, tile, m, n, k):
    """Each tile on shapes that end inside it in every direction, from the
    shortest k on, for every output."""
    w, x, up = codes(1, n, k), codes(2, m, k), codes(3, n, k)
    ws, us, xs = scales(4, n), scales(5, n), scales(6, m, 1e-3, 1e-1)
    y0 = np.random.default_rng(7).standard_normal((m, n)).astype(np.float32)
    y = product(w, ws, x, xs)
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    for ldy in (n, n + 3, (n + 15) // 8 * 8):
        check(run(be, w, ws, x, xs, "f32", ldy), y, "f32")
        check(run(be, w, ws, x, xs, "acc", ldy, y0=y0), y, "acc", y0)
        check(run(be, w, ws, x, xs, "bf16", ldy), y, "bf16")
        check_glu(run(be, w, ws, x, xs, "glu", ldy, up=up, us=us), w, ws, up, us, x, xs)


@pytest.mark.parametrize("tile", ["16x16", "32x16", "48x16", "64x16"])
@pytest.mark.parametrize("m", [1, 9, 16])
def test_weights_read_past_the_caches(be, monkeypatch, tile, m):
    """Up to 16 tokens over 8 MiB of weights and more (4099 x 2048; SwiGLU 2 x
    2051 x 2048), and just below."""
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    for n, f in ((4099, 2051), (4095, 2047)):
        k = 2048
        w, x, up = codes(1, n, k), codes(2, m, k), codes(3, f, k)
        ws, us, xs = scales(4, n, 1e-5, 1e-3), scales(5, f, 1e-5, 1e-3), scales(6, m, 1e-3, 1e-1)
        y0 = np.random.default_rng(7).standard_normal((m, n)).astype(np.float32)
        y = product(w, ws, x, xs)
        check(run(be, w, ws, x, xs, "f32"), y, "f32")
        check(run(be, w, ws, x, xs, "acc", y0=y0), y, "acc", y0)
        check(run(be, w, ws, x, xs, "bf16"), y, "bf16")
        g, gs = np.ascontiguousarray(w[:f]), np.ascontiguousarray(ws[:f])
        check_glu(run(be, g, gs, x, xs, "glu", up=up, us=us), g, gs, up, us, x, xs)


@pytest.mark.parametrize("seed", range(4))
def test_random_shapes(be, monkeypatch, seed):
    """Seeded shapes, outputs, row strides, offsets and tiles (a quarter of them
    the plan's own)."""
    rng = np.random.default_rng(seed)

    def log_int(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))

    for case in range(40):
        m, n, k = log_int(1, 600), log_int(1, 2000), 128 * log_int(2, 24)
        out = rng.choice(["f32", "acc", "bf16", "glu"])
        ldy, offset = n + int(rng.choice([0, 0, 1, 3, 4, 8])), int(rng.choice([0, 0, 4, 8, 2]))
        offset = offset // 4 * 4 if out in ("f32", "acc") else offset
        tile = str(rng.choice(TILES))
        if case % 4:
            monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
        else:
            monkeypatch.delenv("HYMT_HIP_I8_TILE", raising=False)
        w, x, up = codes(case, n, k), codes(case + 1, m, k), codes(case + 2, n, k)
        ws, us, xs = scales(case, n), scales(case + 1, n, 1e-5, 1e-3), scales(case + 2, m, 1e-4, 1e-2)
        y0 = rng.standard_normal((m, n)).astype(np.float32) if out == "acc" else None
        got = run(be, w, ws, x, xs, out, ldy, offset, y0, up, us)
        if out == "glu":
            check_glu(got, w, ws, up, us, x, xs)
        else:
            check(got, product(w, ws, x, xs), out, y0)
