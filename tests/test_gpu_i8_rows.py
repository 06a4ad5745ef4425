"""hymt_to_i8, hymt_rows_rmsnorm_i8 and hymt_weight_i8 on the GPU against numpy
in fp64.  Codes and the sum after an addition are equal: the definition rounds
the exact quotient, and fp32 addition is the same everywhere.  The scale of
to_i8 is one fp64 division rounded to fp32: equal.  The norm's scale is off by
its one rounding to fp32 (half a step) on either side of the reference, whose
sum of squares may be added in another order in fp64 (below 2^-40): 2^-24 (1 + 2^-10)
relative."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from hymt2sharp_amd import synth as S
from tests.i8_cases import U32, Room, bf16_bits, bf16_val, codes_of, norm_rows

pytestmark = pytest.mark.gpu

SHAPES = [(1, 4), (3, 12), (1, 128), (5, 508), (61, 512), (7, 516), (1, 2048), (61, 2048), (6, 2052), (9, 6144),
          (2, 8188), (3, 8192), (700, 2048), (1, 8192)]


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def rows(seed, m, n):
    """Rows of several sizes, with outliers, a row of zeros, rows with a NaN and
    an infinity of either sign, and one of tiny values."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((m, n)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float32)
    x[:, rng.integers(0, n, max(1, n // 300))] *= 20
    if m >= 5:
        x[1] = 0
        x[2, n - 1] = np.nan
        x[3, 0] = -np.inf
        x[4] *= np.float32(1e-37)
    return x


def check(be, got_q, got_s, q, s, tol):
    np.testing.assert_array_equal(got_q, q)
    np.testing.assert_array_equal(np.isnan(got_s), np.isnan(s))
    ok = ~np.isnan(s)
    # below fp32's normal range its steps are 2^-149, a rounding half of one
    assert (np.abs(got_s[ok].astype(np.float64) - s[ok]) <= tol * np.abs(s[ok]) + 2.0 ** -150).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_to_i8(be, m, n, io):
    x = rows(m * 10007 + n, m, n)
    if io == "bf16":
        bits = bf16_bits(np.where(np.isfinite(x), x, 1.0))
        x = np.where(np.isfinite(x), bf16_val(bits), x).astype(np.float32)
        bits = np.where(np.isfinite(x), bits, x.view(np.uint32) >> 16).astype(np.uint16)
    r = Room(be)
    dx = r.put(bits if io == "bf16" else x)
    dq, ds = r.put(np.full((m, n), 55, np.int8)), r.put(np.full(m, -1, np.float32))
    be.to_i8(dx, m, n, dq, ds, x_dtype=N.BF16 if io == "bf16" else N.F32)
    got_q, got_s = r.get(dq, np.empty((m, n), np.int8)), r.get(ds, np.empty(m, np.float32))
    r.close()
    q, a = codes_of(x)
    check(be, got_q, got_s, q, (a / 127.0).astype(np.float32).astype(np.float64), 0.0)


def test_to_i8_ties_go_to_even(be):
    """127 v / a of exactly k + 1/2, for every k: v = (2 k + 1) / 254 of a = 254 d,
    and half of the maximum of bf16 rows."""
    k = np.arange(-127, 127)
    row = ((2 * k + 1) * 0.5).astype(np.float32)  # 127 v / a with a = 127: k + 1/2
    x = np.concatenate([[127.0], row, [0.0]]).astype(np.float32)[None]
    x = np.concatenate([x, x * np.float32(2.0 ** -20), x * np.float32(3), x * np.float32(1.5 * 2.0 ** 40)])
    r = Room(be)
    dx, dq, ds = r.put(x), r.put(np.zeros(x.shape, np.int8)), r.put(np.zeros(4, np.float32))
    be.to_i8(dx, 4, x.shape[1], dq, ds)
    q = r.get(dq, np.empty(x.shape, np.int8))
    b = bf16_bits(np.array([[3.0, 1.5, -1.5, 0.75], [1.0, 0.5, -0.5, 0.25]], np.float32))
    db = r.put(b)
    be.to_i8(db, 2, 4, dq, ds, x_dtype=N.BF16)
    qb = r.get(dq, np.empty((2, 4), np.int8))
    r.close()
    want = np.rint(k + 0.5).astype(np.int8)
    for i in range(4):
        np.testing.assert_array_equal(q[i, 1:-1], want)
    np.testing.assert_array_equal(qb, [[127, 64, -64, 32], [127, 64, -64, 32]])


@pytest.mark.parametrize("add", ["none", "bf16", "f32"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_rows_rmsnorm_i8(be, m, n, add):
    x = rows(m * 131 + n, m, n)
    rng = np.random.default_rng(n)
    w = rng.uniform(-1.2, 1.2, n).astype(np.float32)
    w[rng.integers(0, n)] = 0
    eps = 1e-5
    d = rng.standard_normal((m, n)).astype(np.float32) if add != "none" else None
    if add != "none" and m >= 5:
        d[1] = 0
    dd = None
    r = Room(be)
    if add == "bf16":
        bits = bf16_bits(d)
        d, dd = bf16_val(bits), r.put(bits)
    elif add == "f32":
        dd = r.put(d)
    dx, dw = r.put(x), r.put(w)
    dq, ds = r.put(np.full((m, n), 55, np.int8)), r.put(np.full(m, -1, np.float32))
    be.rows_rmsnorm_i8(dx, m, n, dw, eps, dq, ds, add=dd, add_dtype=N.F32 if add == "f32" else N.BF16)
    got_h = r.get(dx, x)
    got_q, got_s = r.get(dq, np.empty((m, n), np.int8)), r.get(ds, np.empty(m, np.float32))
    r.close()
    h, q, s = norm_rows(x, d, w, eps)
    np.testing.assert_array_equal(got_h, h)
    check(be, got_q, got_s, q, s, U32 * (1 + 2.0 ** -10))


def test_rows_rmsnorm_i8_extremes(be):
    """Values whose squares leave fp32 on either side, eps 0 over a row of
    zeros, weights that make every product zero, and an infinite weight."""
    n = 2048
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, n)).astype(np.float32)
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(1e-30)
    x[2] = 0
    w = np.ones(n, np.float32)
    for kind in ("ones", "zero", "inf"):
        w = {"ones": np.ones, "zero": np.zeros, "inf": np.ones}[kind](n, np.float32)
        if kind == "inf":
            w[5] = np.inf
        r = Room(be)
        dx, dw, dq, ds = r.put(x), r.put(w), r.put(np.full((4, n), 9, np.int8)), r.put(np.zeros(4, np.float32))
        be.rows_rmsnorm_i8(dx, 4, n, dw, 0.0, dq, ds)
        got_q, got_s = r.get(dq, np.empty((4, n), np.int8)), r.get(ds, np.empty(4, np.float32))
        r.close()
        with np.errstate(invalid="ignore"):
            h, q, s = norm_rows(x, None, w, 0.0)
        if kind == "inf":
            assert np.isnan(got_s).all() and not got_q.any()
        else:
            check(be, got_q, got_s, q, s, U32 * (1 + 2.0 ** -10))


def test_no_rows(be):
    r = Room(be)
    dx = r.put(np.ones(64, np.float32))
    dq, ds = r.put(np.full(64, 3, np.int8)), r.put(np.full(1, 7, np.float32))
    be.to_i8(dx, 0, 64, dq, ds)
    be.rows_rmsnorm_i8(dx, 0, 64, dx, 1e-5, dq, ds)
    assert (r.get(dq, np.empty(64, np.int8)) == 3).all() and r.get(ds, np.empty(1, np.float32))[0] == 7
    r.close()


@pytest.mark.parametrize("size", [1.0, 2.0 ** -60, 2.0 ** -100, 2.0 ** 110])
def test_codes_next_to_a_border(be, size):
    """Rows of values within two fp32 steps of every border between two codes,
    of many maxima, in the ranges of both ways to the code."""
    rng = np.random.default_rng(5)
    m, n = 300, 5 * 254 + 2
    a = (rng.uniform(1, 2, m) * size).astype(np.float32)
    mid = (a[:, None].astype(np.float64) * (2 * np.arange(-127, 127) + 1) / 254).astype(np.float32)
    x = np.zeros((m, n), np.float32)
    steps = [mid]
    for to in (np.inf, -np.inf):
        one = np.nextafter(mid, np.float32(to))
        steps += [one, np.nextafter(one, np.float32(to))]
    x[:, :5 * 254] = np.concatenate(steps, 1)
    x[:, -2] = a
    x = np.where(np.abs(x) > a[:, None], np.copysign(a[:, None], x), x)
    w = rng.uniform(0.5, 1.5, n).astype(np.float32)
    near = rng.uniform(0.5, 1.5, (m, 1)).astype(np.float32) * x  # times w: other borders
    r = Room(be)
    dx, dn, dw = r.put(x), r.put(near), r.put(w)
    dq, ds = r.put(np.zeros((m, n), np.int8)), r.put(np.zeros(m, np.float32))
    be.to_i8(dx, m, n, dq, ds)
    q, a = codes_of(x)
    check(be, r.get(dq, np.empty((m, n), np.int8)), r.get(ds, np.empty(m, np.float32)), q,
          (a / 127.0).astype(np.float32).astype(np.float64), 0.0)
    be.rows_rmsnorm_i8(dn, m, n, dw, 0.0, dq, ds)
    np.testing.assert_array_equal(r.get(dq, np.empty((m, n), np.int8)), norm_rows(near, None, w, 0.0)[1])
    be.rows_rmsnorm_i8(dx, m, n, r.put(np.ones(n, np.float32)), 0.0, dq, ds)  # the same borders through the norm
    np.testing.assert_array_equal(r.get(dq, np.empty((m, n), np.int8)), q)
    r.close()


def test_more_rows_than_one_launch_takes(be):
    """Row counts past the 2^23 of one launch: the rows on either side of the
    border, and the last ones."""
    m, n = (1 << 23) + 6, 4
    x = np.random.default_rng(1).standard_normal((m, n)).astype(np.float32)
    d = bf16_bits(np.random.default_rng(2).standard_normal((m, n)))
    w = np.array([1, 0.5, -2, 1], np.float32)
    r = Room(be)
    dx, dd, dw = r.put(x), r.put(d), r.put(w)
    dq, ds = r.put(np.zeros((m, n), np.int8)), r.put(np.zeros(m, np.float32))
    at = np.r_[0:8, (1 << 23) - 8:m]
    be.to_i8(dx, m, n, dq, ds)
    q, a = codes_of(x[at])
    check(be, r.get(dq, np.empty((m, n), np.int8))[at], r.get(ds, np.empty(m, np.float32))[at], q,
          (a / 127.0).astype(np.float32).astype(np.float64), 0.0)
    be.rows_rmsnorm_i8(dx, m, n, dw, 1e-5, dq, ds, add=dd)
    h, q, s = norm_rows(x[at], bf16_val(d[at]), w, 1e-5)
    np.testing.assert_array_equal(r.get(dx, x)[at], h)
    check(be, r.get(dq, np.empty((m, n), np.int8))[at], r.get(ds, np.empty(m, np.float32))[at], q, s,
          U32 * (1 + 2.0 ** -10))
    r.close()


@pytest.mark.parametrize("wtype,rows_,cols", [(N.W_Q4_K, 40, 2048), (N.W_Q6_K, 17, 6144), (N.W_Q8_0, 5, 4096),
                                              (N.W_F32, 9000, 2048), (N.W_F16, 3, 8192)])
def test_weight_i8(be, wtype, rows_, cols):
    """The codes of the dequantized rows, as embed_rows gives them, over more
    than one chunk of them (9000 x 2048)."""
    raw = S.random_weight(7, wtype, rows_, cols)
    w = be.weight_upload(wtype, rows_, cols, raw)
    p = be.alloc(rows_ * cols * 4)
    try:
        be.embed_rows(w, np.arange(rows_), p)
        v = be.download(np.empty((rows_, cols), np.float32), p)
        with pytest.raises(N.InvalidOperationError):
            be.weight_i8_data(w)
        before = be.weight_info(w)["device_bytes"]
        be.weight_i8(w)
        be.weight_i8(w)  # once is enough
        assert be.weight_info(w)["device_bytes"] == before + rows_ * (cols + 4)
        dq, ds = be.weight_i8_data(w)
        got_q = be.download(np.empty((rows_, cols), np.int8), dq)
        got_s = be.download(np.empty(rows_, np.float32), ds)
    finally:
        be.free(p)
        be.weight_free(w)
    q, a = codes_of(v)
    check(be, got_q, got_s, q, (a / 127.0).astype(np.float32).astype(np.float64), 0.0)
