"""The codes of hymt_rows_rmsnorm_i8 where fp64 cannot decide them: products
x * norm_w of 48 bits whose quotient 127 x w / max|x w| is half a code exactly, or
2^-49 to 2^-42 of a code beside it.  The inputs are whole numbers below 2^24 times
a power of two, so the codes follow from whole-number arithmetic."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.i8_cases import Room

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def whole_codes(x, w):
    """rint(127 t / a), ties to even, of t = x w for whole x [m][n] and w [n] below
    2^24: |q| is the largest whole number with (2 q - 1) a <= 254 |t|, less one
    where that is an equality and q is odd.  254 |t| + a is below 2^57."""
    t = np.asarray(x, np.int64) * np.asarray(w, np.int64)
    a = np.abs(t).max(1, keepdims=True)
    num = 254 * np.abs(t) + a
    q = num // (2 * a)
    q -= (num % (2 * a) == 0) & (q % 2 == 1)
    return (np.sign(t) * q).astype(np.int8)


def beside_borders(seed, count):
    """(x0, w0, x, w, r): 254 x w = (2 k + 1) x0 w0 + r for some k below 127 and a
    whole r, 0 < |r| < 16: x w lies |r| / (2 x0 w0) of a code beside the border
    between k and k + 1 of a row whose maximum is x0 w0."""
    rng = np.random.default_rng(seed)
    out = []
    while len(out) < count:
        k, w, w0, r = (int(v) for v in (rng.integers(0, 127), rng.integers(1 << 20, 1 << 24),
                                        rng.integers(1 << 23, 1 << 24), rng.choice([-1, 1]) * rng.integers(1, 16)))
        a, b = 254 * w, (2 * k + 1) * w0
        if np.gcd(a, b) != 1:
            continue
        x = r * pow(a, -1, b) % b
        x0 = (a * x - r) // b
        if 0 < x < 1 << 24 and 1 << 22 < x0 < 1 << 24 and x * w <= x0 * w0:
            assert 254 * x * w == (2 * k + 1) * x0 * w0 + r
            out.append((x0, w0, x, w, r))
    return out


def codes(be, x, w, add, size):
    """The call's codes of x * size (two powers of two: of x and of w) with the
    rows given whole, or as an addition that leaves them."""
    m, n = x.shape
    x = (x * size[0]).astype(np.float32)
    r = Room(be)
    zero = np.zeros((m, n), np.float32)
    dx = r.put(zero if add == "f32" else x)
    dd = r.put(x) if add == "f32" else r.put(np.zeros((m, n), np.uint16)) if add == "bf16" else None
    dw = r.put((w * size[1]).astype(np.float32))
    dq, ds = r.put(np.full((m, n), 55, np.int8)), r.put(np.zeros(m, np.float32))
    be.rows_rmsnorm_i8(dx, m, n, dw, 0.0, dq, ds, add=dd, add_dtype=N.F32 if add == "f32" else N.BF16)
    q = r.get(dq, np.empty((m, n), np.int8))
    r.close()
    return q


SIZES = [(1.0, 1.0), (2.0 ** -60, 2.0 ** -12), (2.0 ** -100, 2.0 ** -80), (2.0 ** 70, 2.0 ** 20)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("add", ["none", "bf16", "f32"])
def test_pairs_under_one_weight(be, add, size):
    """x and x / 2 under one weight: 63.5 goes to 64, and -63.5 to -64, whatever
    the bits of x and the weight."""
    m, n = 200, 2048
    rng = np.random.default_rng(1)
    w = rng.integers(1 << 23, 1 << 24, n)
    w[1::2] = w[::2]
    w[2 * m:] = 1
    x = np.zeros((m, n), np.int64)
    i = np.arange(m)
    x[i, 2 * i] = 2 * rng.integers(1 << 22, 1 << 23, m)
    x[i, 2 * i + 1] = x[i, 2 * i] // 2 * np.where(i % 2, -1, 1)
    want = whole_codes(x, w)
    assert (want[i, 2 * i] == 127).all() and (np.abs(want[i, 2 * i + 1]) == 64).all()
    np.testing.assert_array_equal(codes(be, x, w, add, size), want)


@pytest.mark.parametrize("n", [512, 1024, 2048, 6144])
def test_every_tie(be, n):
    """Half codes of every k under weights of 24 bits: x = 254 d, (2 k + 1) d."""
    m = 50
    rng = np.random.default_rng(n)
    w = np.full(n, int(rng.integers(1 << 23, 1 << 24)))
    d = rng.integers(1 << 15, 1 << 16, (m, 1))
    x = np.zeros((m, n), np.int64)
    x[:, 1:255] = d * (2 * np.arange(-127, 127) + 1)
    x[:, n - 1:] = 254 * d
    want = whole_codes(x, w)
    np.testing.assert_array_equal(want[:, 1:255], np.broadcast_to(np.rint(np.arange(-127, 127) + 0.5), (m, 254)))
    np.testing.assert_array_equal(codes(be, x, w, "none", (1.0, 1.0)), want)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [1024, 4096])
def test_beside_every_border(be, n, size):
    """Values too near to a border for the fp64 quotient, on either side of it."""
    cases = beside_borders(n, 300)
    # the row whose quotient, 115.5 - 2^-47.3, fp64 rounds to a half and to 116
    cases.append((16700629, 15929817, 15418812, 15691735, -3))
    m = n // 2
    cases = [cases[-1 - i % len(cases)] for i in range(m)]
    x, w = np.zeros((m, n), np.int64), np.zeros(n, np.int64)
    for i, (x0, w0, x1, w1, _) in enumerate(cases):
        w[2 * i], w[2 * i + 1] = w0, w1
        x[i, 2 * i], x[i, 2 * i + 1] = x0 * (-1) ** (i % 3), x1 * (-1) ** (i % 2)
    want = whole_codes(x, w)
    assert want[0, 1] == 115
    np.testing.assert_array_equal(codes(be, x, w, "none", size), want)


def test_few_bits(be):
    """Rows and weights of few bits, where ties are common."""
    rng = np.random.default_rng(9)
    for m, n in ((300, 128), (100, 2048)):
        x, w = rng.integers(-400, 401, (m, n)), rng.integers(1, 300, n)
        np.testing.assert_array_equal(codes(be, x, w, "none", (1.0, 2.0 ** -7)), whole_codes(x, w))
