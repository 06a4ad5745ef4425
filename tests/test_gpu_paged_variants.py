"""The forms that the attention over the multi-sequence cache takes by the size of a
batch -- tiles of 64 and of 128 rows, one group of waves or two, ranges cut or whole,
joined by row or by tile, prefixes in either tile -- against the same reference, with
values that are not finite among them."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import PAGE, attention, check_rows, to_bits
from tests.test_gpu_paged_attn import behind, call, cu_of, held, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def longest(c):
    return int(c.len.max())


PACKED = {
    # name: (rows of each entry, lengths, head dim, kv heads, group)
    "64 rows": ([70, 1, 33], [70, 64, 400], 128, 2, 4),
    "64 rows, two groups of waves": ([600, 513, 3], [600, 900, 700], 64, 1, 4),
    "64 rows, two groups, an odd number of pages": ([700], [700], 128, 1, 2),
    "128 rows": ([20 + i % 13 for i in range(70)], [20 + i % 13 + (i % 5) * 30 for i in range(70)], 64, 4, 8),
    "128 rows, one or two pages": ([33] * 80, [33] * 40 + [97] * 40, 128, 4, 3),
    "128 rows, two groups": ([610], [610], 64, 1, 64),
    "cut": ([40, 30], [3000, 2500], 128, 1, 8),
    "cut, groups that end inside a tile": ([19, 5, 50], [2400, 2400, 70], 64, 2, 7),
    "cut into 64": ([3], [6000], 64, 1, 2),
}


@pytest.mark.parametrize("name", PACKED)
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_packed(be, name, dt):
    new, lens, d, hkv, group = PACKED[name]
    c, slots = held(len(name), lens, d=d, kv_heads=hkv, dt=dt)
    run(be, c, slots, cu_of(new), hkv * group, pad=3, max_len=longest(c))


@pytest.mark.parametrize("bad", ["k_nan", "v_nan", "v_inf"])
@pytest.mark.parametrize("rows,length", [(650, 650), (90, 2200), (200, 520)])
def test_packed_with_values_that_are_not_finite(be, bad, rows, length):
    """Two groups of waves, and a range that is cut: rows before a NaN are as
    without it."""
    c, slots = held(3, [length], kv_heads=1, dt=N.BF16)
    s = slots[0]
    x = np.float32(np.nan if bad.endswith("nan") else np.inf)
    pool, off = (c.k, c.ko) if bad[0] == "k" else (c.v, c.vo)
    first = length - rows
    for p, d in ((length - 5, 3), (first + rows // 2, 127), (first + rows // 3, 64)):
        pool[0, c.table[s, p // PAGE], 0, off[p % PAGE, d]] = to_bits(np.array([x]), c.dt)[0]
    before, got, q = call(be, c, slots, [0, rows], 4, max_len=length)
    with np.errstate(invalid="ignore"):
        want, tol, done = attention(c, 0, slots, [0, rows], q, 4)
        check_rows(got, want, np.nan_to_num(tol, nan=0, posinf=0), done, before, c.dt)
    assert np.isfinite(want[:rows // 3]).all() and not np.isfinite(want[rows // 3:]).all(1).any()


SHARED = {
    # name: (slots, prefix, own positions of each, head dim, kv heads, group)
    "by rows": (5, 512, [1, 9, 64, 65, 200], 128, 2, 4),
    "by rows, 20 pages": (5, 1216, [1, 9, 64, 63, 2], 64, 2, 4),
    "64 rows, a page a part": (5, 512, [1, 9, 64, 65, 1500], 128, 2, 4),
    "64 rows, many parts": (3, 4096, [700, 1, 64], 64, 1, 4),
    "128 rows": (66, 8256, [1 + i for i in range(66)], 64, 1, 16),
    "no prefix, cut": (2, 0, [3000, 10], 128, 1, 4),
    "no prefix, whole": (40, 0, [1 + 7 * i for i in range(40)], 64, 8, 3),
    "groups of more than 16 heads": (3, 256, [5, 70, 1], 64, 1, 40),
    "groups of more than 16 heads, in tiles": (3, 256, [5, 70, 1400], 64, 1, 40),
    "groups of more than 16 heads, no prefix": (3, 0, [5, 700, 1], 128, 2, 17),
    "many parts of many rows": (24, 2048, [30] * 24, 64, 4, 16),
}


@pytest.mark.parametrize("name", SHARED)
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_shared(be, name, dt):
    n, prefix, own, d, hkv, group = SHARED[name]
    c, slots = behind(len(name), n, prefix, own, d=d, kv_heads=hkv, dt=dt)
    run(be, c, slots, None, hkv * group, prefix=prefix, max_len=longest(c))


def test_shared_tiles_with_values_that_are_not_finite(be):
    """Slots that end inside the prefix, at lengths spread over a tile of 128 rows."""
    c, slots = behind(5, 66, 8256, [1] * 66, d=64, kv_heads=1, dt=N.BF16)
    for i in range(1, 66, 3):
        c.len[slots[i]] = 8256 - 100 * i
    c.v[0, c.table[slots[0], 60], 0, c.vo[17, 5]] = to_bits(np.array([np.nan], np.float32), c.dt)[0]
    before, got, q = call(be, c, slots, None, 16, prefix=8256, max_len=8257)
    with np.errstate(invalid="ignore"):
        want, tol, done = attention(c, 0, slots, None, q, 16, prefix=8256)
        check_rows(got, want, np.nan_to_num(tol, nan=0, posinf=0), done, before, c.dt)
    sees = np.array([c.len[s] > 60 * 64 + 17 for s in slots])
    assert sees.any() and not sees.all()
    assert (np.isnan(want).any(1) == sees).all()


def test_a_thousand_slots(be):
    own = [1 + i % 70 for i in range(1024)]
    c, slots = behind(6, 1024, 128, own, d=64, kv_heads=1, dt=N.F16, blocks=30)
    run(be, c, slots, None, 2, prefix=128, max_len=longest(c))
    run(be, c, slots, None, 2, prefix=128)  # in tiles
    new = [min(x, 1 + i % 3) for i, x in enumerate(own)]
    run(be, c, slots, cu_of(new), 2, max_len=longest(c))
