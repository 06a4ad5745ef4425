"""hymt_rope_append on the GPU against its formulas in 64 bits (tests/paged_cases.py
derives the tolerances)."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend, Rope, rope_freqs
from hymt2sharp_amd import _native as N
from tests.paged_cases import PAGE, TINY, U, Cache, Room, batch, blocks_of, from_bits, rotated, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def store(a, io):
    return np.ascontiguousarray(a, np.float32) if io == N.F32 else to_bits(a, io)


def value(a, io):
    return a if io == N.F32 else from_bits(a, io)


def run(be, c, slots, cu, heads, io=N.F32, dim=None, interleaved=0, scaling=N.ROPE_NONE, norm=(True, True), pad=0, layer=0,
        seed=0, fused=True, x=None, eps=1e-6, max_len=0):
    """One call, every output checked whole: q rows, both pools, guard bytes."""
    d, hkv = c.d, c.kv_heads
    dim = d if dim is None else dim
    rng = np.random.default_rng(seed)
    total = cu[-1] if cu is not None else len(slots)
    rows = total + pad
    x = rng.standard_normal((max(rows, 1), heads + 2 * hkv, d)) * 2 if x is None else x
    x = store(x, io)
    qw, kw = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2))
    freq, scale = rope_freqs(dim, 10000.0, scaling, 4.0, 4096) if dim else (np.zeros(1), 1.0)
    room = Room(be)
    dev = c.put(room)
    b = batch(room, slots, cu, rows=rows if cu is not None else None, max_len=max_len)
    r = Rope(freq=room.put(freq), dim=dim, interleaved=interleaved, scale=scale)
    es = x.itemsize
    if fused:  # q, k and v as columns of one projection's rows, and 8 values more
        wide = np.concatenate([x.reshape(x.shape[0], -1), np.zeros((x.shape[0], 8), x.dtype)], 1)
        pq = room.put(wide)
        pk, pv, ld = pq + heads * d * es, pq + (heads + hkv) * d * es, (heads + 2 * hkv) * d + 8
        lds = (ld, ld)
    else:
        pq, pk, pv = (room.put(x[:, a:e].reshape(x.shape[0], -1)) for a, e in
                      ((0, heads), (heads, heads + hkv), (heads + hkv, heads + 2 * hkv)))
        lds = (heads * d, hkv * d)
    before = rng.integers(0, 1 << 16, (max(rows, 1), heads * d), dtype=np.uint16)
    out = room.put(before)
    be.rope_append(dev, layer, b, pq, lds[0], pk, pv, lds[1], io, heads, r, room.put(qw) if norm[0] else None,
                   room.put(kw) if norm[1] else None, eps, out)
    got_q = room.get(out, before)
    got_k, got_v = c.get(room, dev, "k", "v")
    ints = c.get(room, dev, "table", "len", "refs", "work")
    room.close()
    for a, w in zip(ints, (c.table, c.len, c.refs, c.work)):
        np.testing.assert_array_equal(a, w)

    xv = value(x, io)[:total].astype(np.float64)
    pos = np.zeros(total, np.int64)
    where = []
    for e, s in enumerate(slots):
        a, z = (e, e + 1) if cu is None else (cu[e], cu[e + 1])
        for i in range(a, z):
            known = 0 <= s < c.seqs
            pos[i] = (int(c.len[s]) if known else 0) - (z - a) + i - a
            page = c.table[s, pos[i] // PAGE] if known and 0 <= pos[i] < c.blocks * PAGE else -1
            if 0 <= page < c.pages:
                where.append((i, int(page), int(pos[i]) % PAGE))

    def near(got, want, err):
        dt = c.dt
        g = from_bits(got, dt).astype(np.float64)
        nan = np.isnan(want)
        np.testing.assert_array_equal(np.isnan(g), nan)
        tol = U[dt] * np.abs(want) + err * (1 + U[dt]) + TINY[dt]
        with np.errstate(invalid="ignore"):
            bad = ~nan & ~(np.abs(g - want) <= tol) & ~(g == want)
        assert not bad.any(), (np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4], tol[bad][:4])

    with np.errstate(invalid="ignore", over="ignore"):
        q, qe = rotated(xv[:, :heads], pos, freq, scale, dim, interleaved, qw if norm[0] else None, eps)
        k, ke = rotated(xv[:, heads:heads + hkv], pos, freq, scale, dim, interleaved, kw if norm[1] else None, eps)
    near(got_q[:total], q.reshape(total, heads * d), qe.reshape(total, heads * d))
    np.testing.assert_array_equal(got_q[total:], before[total:])
    k_at, v_at = c.k.copy(), c.v.copy()
    vb = to_bits(xv[:, heads + hkv:].astype(np.float32), c.dt)
    for i, page, t in where:
        gk = got_k[layer, page][:, c.ko[t]]
        near(gk, k[i], ke[i])
        k_at[layer, page][:, c.ko[t]] = gk
        v_at[layer, page][:, c.vo[t]] = vb[i]
    np.testing.assert_array_equal(got_k, k_at)
    nan = np.isnan(from_bits(v_at, c.dt)) & np.isnan(from_bits(got_v, c.dt))
    np.testing.assert_array_equal(np.where(nan, 0, got_v), np.where(nan, 0, v_at))
    return got_q, got_k, got_v


def held(seed, new, lens, **kw):
    """A cache whose slots (in another order) end with `new` rows each."""
    n = len(new)
    kw.setdefault("seqs", n + 2)
    kw.setdefault("blocks", blocks_of(max(lens)) + 1)
    kw.setdefault("pages", sum(blocks_of(x) for x in lens) + 3)
    c = Cache(seed, **kw)
    slots = np.random.default_rng(seed).permutation(kw["seqs"])[:n].tolist()
    for s, x in zip(slots, lens):
        c.give(s, x, values=False)
    return c, slots, [0] + np.cumsum(new).tolist()


# rows behind the last entry's: few, and so many that the batch goes by blocks of positions
PADS = [3, 1600]
LENGTHS = [([1], [1]), ([5, 0, 1, 64], [5, 0, 1, 64]), ([33, 2, 63], [40, 66, 127]), ([130, 1, 31], [200, 65, 64]),
           ([200], [263])]


@pytest.mark.parametrize("new,lens", LENGTHS)
@pytest.mark.parametrize("d,hkv,group", [(128, 4, 4), (64, 3, 1), (128, 1, 7), (64, 2, 16)])
@pytest.mark.parametrize("pad", PADS)
def test_lengths_and_heads(be, new, lens, d, hkv, group, pad):
    c, slots, cu = held(len(new) * 7 + d, new, lens, d=d, kv_heads=hkv, layers=2)
    run(be, c, slots, cu, hkv * group, pad=pad, layer=1)


@pytest.mark.parametrize("n", [1, 3, 64, 65, 200])
@pytest.mark.parametrize("d,dt", [(128, N.BF16), (64, N.F16)])
def test_one_row_each(be, n, d, dt):
    lens = np.random.default_rng(n).integers(1, 400, n).tolist()
    c, slots, _ = held(n, [1] * n, lens, d=d, dt=dt)
    run(be, c, slots, None, 8)


@pytest.mark.parametrize("io", [N.F32, N.F16, N.BF16])
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
@pytest.mark.parametrize("fused", [True, False])
def test_types_and_strides(be, io, dt, fused):
    c, slots, cu = held(3, [40, 70], [100, 70], dt=dt, kv_heads=2)
    for pad in PADS:
        run(be, c, slots, cu, 6, io=io, fused=fused, pad=pad)
    run(be, c, slots, None, 6, io=io, fused=fused)


@pytest.mark.parametrize("d,dim", [(128, x) for x in (0, 16, 32, 48, 64, 96, 112, 128)] + [(64, x) for x in (0, 16, 48, 64)])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("pad", PADS)
def test_rotated_part(be, d, dim, interleaved, pad):
    c, slots, cu = held(dim, [50, 9], [77, 9], d=d, dt=N.F16)
    run(be, c, slots, cu, 4, dim=dim, interleaved=interleaved, pad=pad)


@pytest.mark.parametrize("scaling", [N.ROPE_LINEAR, N.ROPE_NTK, N.ROPE_YARN])
@pytest.mark.parametrize("norm", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("pad", PADS)
def test_scalings_and_norms(be, scaling, norm, pad):
    c, slots, cu = held(9, [20, 3], [50, 300], dt=N.F16)
    run(be, c, slots, cu, 4, scaling=scaling, norm=norm, pad=pad)


@pytest.mark.parametrize("n,rows", [(1, 1535), (1, 1536), (3, 800), (120, 13), (120, 14), (120, 15)])
def test_many_rows(be, n, rows):
    """Both sides of where a batch goes by blocks, entries at every offset in a page."""
    new = [max(rows + (i % 3 - 1) * (n > 2), 0) for i in range(n)]
    c, slots, cu = held(n + rows, new, [x + 7 * i % 130 for i, x in enumerate(new)], kv_heads=1, d=64)
    run(be, c, slots, cu, 2)


def test_far_positions(be):
    """Angles of positions up to 10^6 (in fp32 the product with the frequency alone
    would be off by 0.03 radians)."""
    c = Cache(1, pages=4, seqs=3, blocks=1 << 14, dt=N.F16)
    for s, p in ((0, 1 << 20), (1, 999983), (2, 524289)):
        c.len[s] = p
        c.table[s, (p - 1) // PAGE] = s
        c.refs[s] = 1
    run(be, c, [2, 0, 1], None, 4)


def test_rows_of_zeros_infinities_and_nan(be):
    c, slots, cu = held(4, [70], [70], dt=N.BF16)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((70, 4 + 4, 128)).astype(np.float32)
    x[3] = 0
    x[5, 2, 7] = np.nan
    x[6, 5] = np.nan
    x[9, 6, 3] = np.inf
    x[10, 7, 100] = -np.inf
    for more in (0, 1600):
        wide = np.concatenate([x, np.zeros((more, 8, 128), np.float32)])
        run(be, c, slots, cu, 4, x=wide, norm=(False, False), dim=0, pad=more)
        run(be, c, slots, cu, 4, x=np.where(np.isinf(wide), np.nan, wide), pad=more)


def test_slots_and_pages_that_are_not_there(be):
    """Rows of an unknown slot, before position 0, past the table, and of pages outside
    the pool: q is written, k and v nowhere."""
    c, slots, cu = held(6, [10, 70, 4], [100, 70, 4], seqs=5)
    c.table[slots[1], 0] = -1
    c.table[slots[0], 1] = c.pages
    c.len[slots[2]] = 2  # two of its four rows stand before position 0
    for pad in PADS:
        run(be, c, slots + [-1, 5, 1 << 30], cu + [cu[-1] + 2, cu[-1] + 3, cu[-1] + 3], 4, pad=pad)


def test_nothing_to_do(be):
    c, slots, cu = held(6, [0, 0], [10, 0])
    run(be, c, slots, cu, 4)
    run(be, c, slots, cu, 4, pad=5)
    run(be, c, slots, cu, 4, pad=1600)


def test_a_row_has_the_same_bits_in_every_batch(be):
    """Alone, among others, packed or one by one."""
    c, slots, cu = held(8, [1, 1, 1], [100, 5, 64])
    x = np.random.default_rng(1).standard_normal((3, 12, 128)).astype(np.float32)
    q0, k0, v0 = run(be, c, slots, None, 8, x=x)
    q1, k1, v1 = run(be, c, slots, cu, 8, x=x)
    np.testing.assert_array_equal(q0, q1)
    np.testing.assert_array_equal(k0, k1)
    np.testing.assert_array_equal(v0, v1)
    wide = np.concatenate([x, np.zeros((1600, 12, 128), np.float32)])
    q3, k3, v3 = run(be, c, slots, cu, 8, x=wide, pad=1600)
    np.testing.assert_array_equal(q0, q3[:3])
    np.testing.assert_array_equal(k0, k3)
    np.testing.assert_array_equal(v0, v3)
    q2, _, _ = run(be, c, slots[1:2], None, 8, x=x[1:2])
    np.testing.assert_array_equal(q2[0], q0[1])
