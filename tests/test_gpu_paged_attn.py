"""hymt_attn_packed and hymt_attn_shared on the GPU against softmax(q K^T) V in 64
bits (tests/paged_cases.py derives the tolerances).  Positions that nothing may
read hold random bits, NaN and infinities among them."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import PAGE, Cache, Room, attention, batch, blocks_of, check_rows, from_bits, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def held(seed, lens, extra=3, **kw):
    n = len(lens)
    kw.setdefault("seqs", n + 2)
    kw.setdefault("blocks", blocks_of(max(list(lens) + [1])) + 1)
    kw.setdefault("pages", sum(blocks_of(x) for x in lens) + extra)
    c = Cache(seed, **kw)
    slots = np.random.default_rng(seed).permutation(kw["seqs"])[:n].tolist()
    for s, x in zip(slots, lens):
        c.give(s, x)
    return c, slots


def call(be, c, slots, cu, heads, q=None, layer=0, scale=None, out_dt=None, pad=0, prefix=None, max_len=0, seed=0):
    """(bits of out before and after, q values): one call, inputs and guards unchanged."""
    rng = np.random.default_rng(seed + 1)
    rows = (cu[-1] if cu is not None else len(slots)) + pad
    if q is None:
        q = rng.standard_normal((max(rows, 1), heads * c.d))
    qb = to_bits(q, c.dt)
    before = rng.integers(0, 1 << 16, (max(rows, 1), heads * c.d), dtype=np.uint16)
    room = Room(be)
    dev = c.put(room)
    b = batch(room, slots, cu, rows=rows if cu is not None else None, max_len=max_len)
    dq, out = room.put(qb), room.put(before)
    if prefix is None:
        be.attn_packed(dev, layer, b, dq, heads, out, scale=scale, out_dtype=out_dt)
    else:
        be.attn_shared(dev, layer, b, prefix, dq, heads, out, scale=scale, out_dtype=out_dt)
    got = room.get(out, before)
    for name, a in zip(("k", "v", "table", "len", "refs"), c.get(room, dev, "k", "v", "table", "len", "refs")):
        np.testing.assert_array_equal(a, getattr(c, name), err_msg=name)
    np.testing.assert_array_equal(room.get(dq, qb), qb)
    room.close()
    return before, got, from_bits(qb, c.dt)


def run(be, c, slots, cu, heads, layer=0, scale=None, out_dt=None, prefix=None, **kw):
    before, got, q = call(be, c, slots, cu, heads, layer=layer, scale=scale, out_dt=out_dt, prefix=prefix, **kw)
    want, tol, done = attention(c, layer, slots, cu, q, heads, scale, prefix or 0, out_dt)
    check_rows(got, want, tol, done, before, c.dt if out_dt is None else out_dt)
    return got


def cu_of(new):
    return [0] + np.cumsum(new).tolist()


HEADS = [(128, 4, 4), (128, 2, 1), (64, 3, 5), (64, 1, 16), (128, 1, 7), (64, 8, 2)]


# ---- packed ------------------------------------------------------------------------

PACKED = [([1], [1]), ([64], [64]), ([65], [65]), ([3, 0, 1, 130], [3, 0, 1, 130]), ([31, 33, 2], [31, 97, 66]),
          ([7, 128, 1], [200, 320, 65]), ([150, 0, 0], [150, 5, 0])]


@pytest.mark.parametrize("new,lens", PACKED)
@pytest.mark.parametrize("d,hkv,group", HEADS)
def test_packed(be, new, lens, d, hkv, group):
    dt = N.F16 if (d + len(new)) % 3 else N.BF16
    c, slots = held(len(new) + d + group, lens, d=d, kv_heads=hkv, dt=dt, layers=2)
    run(be, c, slots, cu_of(new), hkv * group, pad=4, layer=1)


@pytest.mark.parametrize("dt", [N.F16, N.BF16])
@pytest.mark.parametrize("out_dt", [N.F16, N.BF16])
def test_packed_types_and_scales(be, dt, out_dt):
    c, slots = held(5, [100, 70], dt=dt)
    for scale in (None, 1.0, 0.0, -0.2):
        run(be, c, slots, cu_of([100, 9]), 8, scale=scale, out_dt=out_dt)


def test_packed_long(be):
    """More tiles than a workgroup's ring, ragged, over many pages in any order."""
    c, slots = held(2, [900, 1, 451], kv_heads=1, dt=N.BF16)
    run(be, c, slots, cu_of([300, 1, 451]), 2, pad=1)


@pytest.mark.parametrize("max_len", [0, 1, 3000, 1 << 30])
def test_packed_few_rows_over_many_positions(be, max_len):
    """The split of a long cache and its joining, whatever the caller says of the
    lengths."""
    c, slots = held(3, [3000, 2100, 64], kv_heads=2, dt=N.F16)
    run(be, c, slots, cu_of([5, 70, 1]), 8, max_len=max_len)


def test_packed_many_entries(be):
    rng = np.random.default_rng(3)
    new = rng.integers(0, 4, 200).tolist()
    lens = [a + int(x) for a, x in zip(new, rng.integers(0, 70, 200))]
    c, slots = held(4, lens, kv_heads=1, d=64)
    run(be, c, slots, cu_of(new), 4, pad=2)


@pytest.mark.parametrize("n", [1, 64, 65, 300])
@pytest.mark.parametrize("group", [3, 64])
def test_packed_single_rows_without_offsets(be, n, group):
    lens = np.random.default_rng(n).integers(0, 200, n).tolist()
    c, slots = held(n, lens, kv_heads=1, d=64, dt=N.F16)
    run(be, c, slots, None, group)


@pytest.mark.parametrize("lens", [[3000], [5000, 1, 0, 2600, 64], [2900] * 30])
def test_packed_single_rows_over_many_positions(be, lens):
    """Cut and joined, with offsets and without: the same bits."""
    c, slots = held(len(lens), lens, kv_heads=1, d=64, dt=N.F16)
    a = run(be, c, slots, None, 5)
    b = run(be, c, slots, list(range(len(lens) + 1)), 5)
    np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("n", [300, 1024])
def test_packed_hundreds_of_prompts(be, n):
    rng = np.random.default_rng(n)
    new = rng.integers(0, 40, n) * (rng.random(n) < 0.3)
    new[[0, n - 1]] = 0, 33
    lens = (new + rng.integers(0, 70, n)).tolist()
    c, slots = held(5, lens, kv_heads=2, d=64)
    run(be, c, slots, cu_of(new), 10, pad=2)


def test_rows_without_positions(be):
    """Unknown slots, rows before position 0 and empty slots: zeros."""
    c, slots = held(6, [40, 10], seqs=4)
    c.len[slots[1]] = 3
    sl = slots + [-1, 99]
    cu = cu_of([5, 7, 2, 1])
    before, got, q = call(be, c, sl, cu, 8)
    known = attention(c, 0, slots, cu[:3], q[:12], 8)
    check_rows(got[:12], *known, before[:12], c.dt)
    assert (from_bits(got[12:15], c.dt) == 0).all()


@pytest.mark.parametrize("bad", ["k_nan", "k_inf", "v_nan", "v_inf"])
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_what_a_row_does_not_see_does_not_reach_it(be, bad, dt):
    """NaN and infinities at positions 40, 70 and 150: rows before them are as
    without them, rows that see one have the formula's value."""
    c, slots = held(7, [200], kv_heads=2, dt=dt)
    s = slots[0]
    x = np.float32(np.nan if bad.endswith("nan") else np.inf)
    pool, off = (c.k, c.ko) if bad[0] == "k" else (c.v, c.vo)
    for p, d in ((70, 5), (150, 127), (40, 64)):
        if p == 40 and bad[0] == "k":
            continue
        pool[0, c.table[s, p // PAGE], 1, off[p % PAGE, d]] = to_bits(np.array([x]), dt)[0]
    q = np.abs(np.random.default_rng(1).standard_normal((200, 8 * 128)))
    q[::2] *= -1  # an infinite key: scores of either sign
    before, got, qv = call(be, c, slots, [0, 200], 8, q=q)
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol, done = attention(c, 0, slots, [0, 200], qv, 8)
        check_rows(got, want, np.nan_to_num(tol, nan=0, posinf=0), done, before, dt)
    sees = 40 if bad[0] == "v" else 70
    assert np.isfinite(want[:sees]).all() and not np.isfinite(want[sees:]).all()


@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_large_and_lopsided_scores(be, dt):
    """Scores of several hundred, a maximum that rises from tile to tile, and one
    position that takes all the weight."""
    c, slots = held(8, [500], kv_heads=1, dt=dt)
    s = slots[0]
    k = np.random.default_rng(2).standard_normal((500, 128)) * np.linspace(0.1, 12, 500)[:, None]
    k[333] = 20
    for p in range(500):
        c.k[0, c.table[s, p // PAGE], 0, c.ko[p % PAGE]] = to_bits(k[p], dt)
    q = np.random.default_rng(3).standard_normal((500, 2 * 128)) * 3
    q[400:] = 1
    run(be, c, slots, [0, 500], 2, q=q)


@pytest.mark.parametrize("form", ["packed", "few_rows", "single", "shared", "shared in tiles"])
@pytest.mark.parametrize("dt,qv,kv", [(N.BF16, 2.0 ** 60, -2.0 ** 62), (N.BF16, 2.0 ** 60, 2.0 ** 61), (N.BF16, 3.0, 2.0 ** 20),
                                      (N.F16, 60000.0, 30000.0), (N.F16, 60000.0, -30000.0)])
@pytest.mark.parametrize("scale", [None, 0.0])
def test_scores_far_from_zero(be, form, dt, qv, kv, scale):
    """Equal scores of up to +-2^126: every weight is 1 and the result the mean of
    V, to the fp32 sums' (n + 8) 2^-24 of the mean of |v| and one rounding; and a position
    that stands out by half a score takes all."""
    lens = [300, 90] if form != "few_rows" else [3000, 90]
    blocks = 80 if form == "shared in tiles" else blocks_of(max(lens)) + 1
    form = form.split()[0]
    c, slots = held(11, lens, kv_heads=1, d=64, dt=dt, blocks=blocks)
    c.k[:] = to_bits(np.full(1, kv / 8), dt)[0]
    new = {"packed": lens, "few_rows": [20, 7], "single": [1, 1], "shared": [1, 1]}[form]
    prefix = 64 if form == "shared" else 0 if form == "single" else None
    if form == "shared":
        c.refs[c.table[slots[0], 0]] += 1
        c.table[slots[1], 0] = c.table[slots[0], 0]
    q = np.full((sum(new), 2 * 64), qv / 8)
    cu = None if prefix is not None else cu_of(new)
    got = call(be, c, slots, cu, 2, q=q, scale=scale, prefix=prefix)[1]
    got = from_bits(got, dt).astype(np.float64).reshape(-1, 2, 64)
    u = 2.0 ** -11 if dt == N.F16 else 2.0 ** -8
    r = 0
    for s, n, length in zip(slots, new, lens):
        v = c.rows(0, s, length)[1][0]
        for j in range(n):
            x = v[:length - n + 1 + j]
            tol = (len(x) + 8) * 2.0 ** -24 * np.abs(x).mean(0) + u * np.abs(x.mean(0)) + 2.0 ** -25
            assert (np.abs(got[r] - x.mean(0)) <= tol).all(), (r, j)
            r += 1
    if scale is None:
        for s in slots:
            c.k[0, c.table[s, 0], 0, c.ko[5]] = to_bits(np.full(1, kv / 8 * (1.5 if kv > 0 else 0.5)), dt)[0]
        got = call(be, c, slots, cu, 2, q=q, prefix=prefix)[1].reshape(-1, 2, 64)
        r = 0
        for s, n, length in zip(slots, new, lens):
            for j in range(n):
                if length - n + j >= 5:
                    assert (got[r] == c.v[0, c.table[s, 0], 0, c.vo[5]]).all(), (r, j)
                r += 1


def test_rows_have_the_same_bits_twice(be):
    c, slots = held(9, [700, 64, 1500], dt=N.F16)
    a = call(be, c, slots, cu_of([100, 64, 20]), 16)[1]
    b = call(be, c, slots, cu_of([100, 64, 20]), 16)[1]
    np.testing.assert_array_equal(a, b)


# ---- shared ------------------------------------------------------------------------


ROOM = [0]


@pytest.fixture(params=["by rows", "in tiles"])
def way(request):
    """Short sequences read their prefix row by row, unless the slots could be long (and
    the batch does not say): then tiles of all rows do."""
    ROOM[0] = 60 if request.param == "in tiles" else 0
    yield
    ROOM[0] = 0


def behind(seed, n, prefix, own, **kw):
    """n slots that begin with the same `prefix` positions, own[i] after them."""
    kw.setdefault("seqs", n + 2)
    kw.setdefault("blocks", blocks_of(prefix + max(own)) + 1 + ROOM[0])
    kw.setdefault("pages", prefix // PAGE + sum(blocks_of(x) for x in own) + 3)
    c = Cache(seed, **kw)
    slots = np.random.default_rng(seed).permutation(kw["seqs"])[:n].tolist()
    for i, (s, x) in enumerate(zip(slots, own)):
        if i == 0 or prefix == 0:
            c.give(s, prefix + x)
            continue
        free = [int(p) for p in np.flatnonzero(c.refs == 0)]
        c.rng.shuffle(free)
        common = c.table[slots[0], :prefix // PAGE].tolist()
        c.give(s, prefix + x, pages=common + free, values=False)
        for b, p in enumerate(free[:blocks_of(x)]):
            m = min(PAGE, x - b * PAGE)
            for pool, off in ((c.k, c.ko), (c.v, c.vo)):
                pool[:, p][:, :, off[:m]] = to_bits(c.rng.standard_normal((c.layers, c.kv_heads, m, c.d)), c.dt)
    return c, slots


@pytest.mark.parametrize("n,prefix,own", [(1, 64, [1]), (3, 64, [1, 64, 65]), (5, 320, [1, 200, 3, 64, 130]),
                                          (2, 0, [1, 300]), (40, 128, [1 + 7 * i % 90 for i in range(40)]),
                                          (9, 1024, [2] * 9)])
@pytest.mark.parametrize("d,hkv,group", HEADS)
@pytest.mark.usefixtures("way")
def test_shared(be, n, prefix, own, d, hkv, group):
    dt = N.F16 if (d + n) % 3 else N.BF16
    c, slots = behind(n + d, n, prefix, own, d=d, kv_heads=hkv, dt=dt, layers=2)
    run(be, c, slots, None, hkv * group, prefix=prefix, layer=1)


@pytest.mark.parametrize("dt", [N.F16, N.BF16])
@pytest.mark.parametrize("out_dt", [N.F16, N.BF16])
@pytest.mark.usefixtures("way")
def test_shared_types_and_scales(be, dt, out_dt):
    c, slots = behind(5, 4, 192, [1, 5, 64, 100], dt=dt)
    for scale in (None, 1.0, 0.0, -0.2):
        run(be, c, slots, None, 8, scale=scale, out_dt=out_dt, prefix=192)


@pytest.mark.parametrize("max_len", [0, 1, 2600, 1 << 30])
def test_shared_long(be, max_len):
    """Prefixes and own parts that are split, and joined in one row."""
    c, slots = behind(3, 4, 1536, [1000, 1, 64, 513], kv_heads=1, dt=N.F16)
    run(be, c, slots, None, 4, prefix=1536, max_len=max_len)
    run(be, c, slots, None, 4, prefix=512, max_len=max_len)
    run(be, c, slots, None, 4, prefix=0, max_len=max_len)


@pytest.mark.usefixtures("way")
def test_shared_many(be):
    own = [1 + (i * 37) % 130 for i in range(300)]
    c, slots = behind(4, 300, 256, own, kv_heads=1, d=64)
    run(be, c, slots, None, 3, prefix=256)


@pytest.mark.usefixtures("way")
def test_shorter_than_the_prefix(be):
    """Slots that end inside the prefix, empty ones, and one that begins otherwise:
    its first positions are read as slots[0]'s."""
    c, slots = behind(6, 6, 256, [10, 20, 30, 40, 1, 1])
    c.len[slots[1]], c.len[slots[2]], c.len[slots[3]] = 100, 0, 256
    c.table[slots[4], 0] = c.table[slots[0], 4]
    run(be, c, slots, None, 8, prefix=256)


@pytest.mark.usefixtures("way")
def test_first_slot_shorter_than_the_prefix(be):
    """Only its whole pages are shared; the others read their own from there on."""
    c, slots = behind(7, 4, 256, [1, 20, 64, 90])
    c.len[slots[0]] = 150
    run(be, c, slots, None, 8, prefix=256)
    c.len[slots[0]] = 0
    run(be, c, slots, None, 8, prefix=256)


@pytest.mark.usefixtures("way")
def test_shared_unknown_slots_and_pages(be):
    c, slots = behind(8, 3, 128, [10, 70, 5])
    sl = [slots[0], -1, slots[1], 77, slots[2]]
    before, got, q = call(be, c, sl, None, 8, prefix=128)
    known = [0, 2, 4]
    want, tol, done = attention(c, 0, slots, None, q[known], 8, prefix=128)
    check_rows(got[known], want, tol, done, before[known], c.dt)
    assert (from_bits(got[[1, 3]], c.dt) == 0).all()
    before, got, _ = call(be, c, [-5] + slots, None, 8, prefix=128)  # the first one unknown: nothing is shared
    np.testing.assert_array_equal(from_bits(got[0], c.dt), 0)


@pytest.mark.usefixtures("way")
def test_pages_outside_the_pool_are_absent(be):
    """A page entry outside the pool hides its positions, in either form."""
    c, slots = behind(9, 2, 128, [70, 70], kv_heads=1)
    hidden = c.table[slots[1], 2]
    q = np.random.default_rng(0).standard_normal((2, 4 * 128))
    for bad in (-1, c.pages, 1 << 30, -(1 << 31)):
        c.table[slots[1], 2] = bad
        for prefix in (128, 0):
            _, got, qv = call(be, c, slots, None, 4, q=q, prefix=prefix)
            _, packed, _ = call(be, c, slots, [0, 1, 2], 4, q=q)
            # positions 128 .. 191 of the second slot are gone: attend to the rest
            c.table[slots[1], 2] = hidden
            k, v = c.rows(0, slots[1], 198)
            seen = np.r_[0:128, 192:198]
            from tests.paged_cases import attend
            for h in range(4):
                col = slice(h * 128, (h + 1) * 128)
                want, tol = attend(qv[1:2, col].astype(np.float64), k[0][seen], v[0][seen], [len(seen)], 128 ** -0.5, c.dt)
                for g in (got, packed):
                    assert (np.abs(from_bits(g[1:2, col], c.dt) - want) <= tol).all()
            c.table[slots[1], 2] = bad
    c.table[slots[1], 2] = hidden


@pytest.mark.parametrize("bad", ["v_nan", "v_inf", "k_nan"])
@pytest.mark.usefixtures("way")
def test_shared_and_values_that_some_rows_do_not_see(be, bad):
    """A slot that ends inside the prefix does not see what stands after it."""
    c, slots = behind(10, 5, 192, [5, 5, 5, 5, 5], kv_heads=1, dt=N.BF16)
    c.len[slots[1]], c.len[slots[3]] = 130, 90
    x = np.float32(np.nan if bad.endswith("nan") else np.inf)
    pool, off = (c.k, c.ko) if bad[0] == "k" else (c.v, c.vo)
    pool[0, c.table[slots[0], 2], 0, off[140 - 128, 9]] = to_bits(np.array([x]), N.BF16)[0]
    before, got, qv = call(be, c, slots, None, 4, prefix=192)
    with np.errstate(invalid="ignore"):
        want, tol, done = attention(c, 0, slots, None, qv, 4, prefix=192)
        check_rows(got, want, np.nan_to_num(tol, nan=0, posinf=0), done, before, c.dt)
    assert np.isfinite(want[[1, 3]]).all() and not np.isfinite(want[0]).all()


@pytest.mark.usefixtures("way")
def test_shared_has_the_same_bits_twice(be):
    c, slots = behind(11, 20, 1024, [1 + 40 * i for i in range(20)], dt=N.F16, kv_heads=2)
    a = call(be, c, slots, None, 16, prefix=1024)[1]
    b = call(be, c, slots, None, 16, prefix=1024)[1]
    np.testing.assert_array_equal(a, b)


def test_offsets_past_2_32(be):
    """The last page of a pool of 5 GB, in its last layer."""
    layers, pages, hkv, d = 40, 2048, 4, 128
    dev = be.paged_create(layers, pages, 2, 3, kv_heads=hkv, head_dim=d, dtype=N.F16)
    room = Room(be)
    try:
        c = Cache(12, layers=1, pages=1, kv_heads=hkv, d=d, dt=N.F16, seqs=2, blocks=3)
        c.give(1, 50)
        page = hkv * PAGE * d * 2
        at = (layers * pages - 1) * page
        assert at > 1 << 32
        be.upload(dev.k + at, c.k)
        be.upload(dev.v + at, c.v)
        be.upload(dev.table, np.array([[-1] * 3, [pages - 1, -1, -1]], np.int32))
        be.upload(dev.len, c.len)
        q = to_bits(np.random.default_rng(0).standard_normal((50, 8 * d)), N.F16)
        before = np.zeros((50, 8 * d), np.uint16)
        out = room.put(before)
        be.attn_packed(dev, layers - 1, batch(room, [1], [0, 50]), room.put(q), 8, out)
        want, tol, done = attention(c, 0, [1], [0, 50], from_bits(q, N.F16), 8)
        check_rows(room.get(out, before), want, tol, done, before, N.F16)
        be.attn_shared(dev, layers - 1, batch(room, [1]), 0, room.put(q[49:]), 8, out)
        check_rows(room.get(out, before)[:1], want[49:], tol[49:], done[49:], before[:1], N.F16)
    finally:
        room.close()
        be.paged_free(dev)
