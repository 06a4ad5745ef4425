"""hymt_paged_extend, _fork, _set_len and _compact on the GPU against the same rules
in plain Python: whole numbers and moved bits, so everything is equal."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import PAGE, Cache, Room, blocks_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


class Model:
    """The rules of include/hymt_hip.h on a Cache's host arrays."""

    def __init__(self, c):
        self.c = c

    def free(self, n):
        f = np.flatnonzero(self.c.refs <= 0)
        return [int(p) for p in f[:n]] if len(f) >= n else None

    def end(self, status, copies=0, live=None):
        w = self.c.work
        w[3], w[1] = status, copies
        if status and not w[0]:
            w[0] = status
        if live is not None:
            w[2] = live

    def extend(self, slots, add):
        c = self.c
        need = [blocks_of(int(c.len[s]) + a) - blocks_of(int(c.len[s])) for s, a in zip(slots, add)]
        pages = self.free(sum(need))
        for s, a, k in zip(slots, add, need):
            b = blocks_of(int(c.len[s]))
            for p in pages[:k]:
                c.table[s, b] = p
                c.refs[p] = 1
                b += 1
            pages = pages[k:]
            c.len[s] += a
        self.end(0)

    def copy(self, pairs):
        for pool in (self.c.k, self.c.v):
            old = pool.copy()
            for a, b in pairs:
                pool[:, b] = old[:, a]

    def fork(self, parent, child):
        c = self.c
        pages = self.free(sum(int(c.len[p]) % PAGE > 0 for p in parent))
        pairs = []
        for p, s in zip(parent, child):
            whole = int(c.len[p]) // PAGE
            c.table[s, :whole] = c.table[p, :whole]
            for b in range(whole):
                c.refs[c.table[p, b]] += 1
            if c.len[p] % PAGE:
                q = pages.pop(0)
                pairs.append((int(c.table[p, whole]), q))
                c.table[s, whole] = q
                c.refs[q] = 1
            c.len[s] = c.len[p]
        self.copy(pairs)
        self.end(0, len(pairs))

    def set_len(self, slots, lens):
        c = self.c
        want = [min(int(c.len[s]), k) for s, k in zip(slots, lens)]
        cut = [s for s, k in zip(slots, want) if k < c.len[s] and k % PAGE and c.refs[c.table[s, k // PAGE]] > 1]
        pages, pairs = self.free(len(cut)), []
        for s, k in zip(slots, want):
            if s in cut:
                q = pages.pop(0)
                old = int(c.table[s, k // PAGE])
                pairs.append((old, q))
        done = iter(pairs)
        for s, k in zip(slots, want):
            if s in cut:
                old, q = next(done)
                c.table[s, k // PAGE] = q
                c.refs[q], c.refs[old] = 1, c.refs[old] - 1
            for b in range(blocks_of(k), blocks_of(int(c.len[s]))):
                c.refs[c.table[s, b]] -= 1
                c.table[s, b] = -1
            c.len[s] = k
        self.copy(pairs)
        self.end(0, len(pairs))

    def compact(self):
        c = self.c
        live = int((c.refs > 0).sum())
        holes = [p for p in range(live) if c.refs[p] <= 0]
        movers = [p for p in range(live, c.pages) if c.refs[p] > 0]
        pairs = list(zip(movers, holes))
        for a, b in pairs:
            c.table[c.table == a] = b
            c.refs[b], c.refs[a] = c.refs[a], 0
        self.copy(pairs)
        self.end(0, len(pairs), live)


def ints(room, v):
    return room.put(np.asarray(v, np.int32))


def offsets_of(add):
    return np.concatenate([[0], np.cumsum(add)]).astype(np.int32)


def equal(c, room, dev):
    table, ln, refs, work, k, v = c.get(room, dev, "table", "len", "refs", "work", "k", "v")
    np.testing.assert_array_equal(table, c.table)
    np.testing.assert_array_equal(ln, c.len)
    np.testing.assert_array_equal(refs, c.refs)
    np.testing.assert_array_equal(work[:4], c.work[:4])
    np.testing.assert_array_equal(k, c.k)
    np.testing.assert_array_equal(v, c.v)


@pytest.mark.parametrize("d,hkv,layers,dt", [(128, 4, 3, N.BF16), (64, 3, 1, N.F16), (128, 1, 2, N.F16)])
def test_a_life_of_sequences(be, d, hkv, layers, dt):
    """Extend, fork, cut, free and compact in turn over the whole range of lengths
    (none, one, a page's end and its neighbours), checked whole after every call."""
    c = Cache(5, layers=layers, pages=150, kv_heads=hkv, d=d, dt=dt, seqs=12, blocks=20)
    m, room = Model(c), Room(be)
    dev = c.put(room)
    steps = [
        ("extend", [3, 0, 7], [200, 64, 1]),
        ("extend", [7, 1], [62, 0]),
        ("extend", [0, 3, 7, 1], [1, 56, 1, 63]),  # to 65, 256, 64, 63
        ("fork", [3, 3, 0, 7], [2, 5, 8, 9]),
        ("extend", [2, 5, 8, 3, 9], [1, 130, 3, 64, 1]),
        ("set_len", [5, 2, 3], [100, 256, 192]),   # inside a page that 3 and 2 hold; at an end; one page back
        ("set_len", [2, 3], [65, 70]),             # both inside the same pages
        ("compact",),
        ("set_len", [8, 0], None),
        ("fork", [5], [0]),
        ("set_len", [5, 0, 9], [1, 9999, 0]),
        ("compact",),
        ("compact",),
        ("extend", [8, 11, 10], [1000, 1, 1279]),
        ("set_len", [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], None),
    ]
    for op, *args in steps:
        if op == "extend":
            be.paged_extend(dev, ints(room, args[0]), len(args[0]), cu=ints(room, offsets_of(args[1])))
            m.extend(*args)
        elif op == "fork":
            be.paged_fork(dev, ints(room, args[0]), ints(room, args[1]), len(args[0]))
            m.fork(*args)
        elif op == "set_len":
            be.paged_set_len(dev, ints(room, args[0]), len(args[0]), lens=None if args[1] is None else ints(room, args[1]))
            m.set_len(args[0], args[1] or [0] * len(args[0]))
        else:
            be.paged_compact(dev)
            m.compact()
        equal(c, room, dev)
    assert (c.refs == 0).all() and be.paged_work(dev)["first"] == 0
    room.close()


@pytest.mark.parametrize("n,pages,seqs", [(1, 3, 1), (64, 700, 70), (1024, 5000, 1500), (300, 70000, 4000)])
def test_many_slots_and_pages(be, n, pages, seqs):
    """One position each, many times the plan's threads of pages, references up
    to 1000, and a pool that is full to the last page."""
    rng = np.random.default_rng(n)
    c = Cache(n, pages=pages, kv_heads=1, d=64, seqs=seqs, blocks=5)
    slots = rng.permutation(seqs)[:n]
    keep = rng.permutation(pages)[:min(n, pages - 2 * n if pages > 2 * n else 1)]
    for s, p in zip(slots, keep):
        c.give(s, int(rng.integers(1, 65)), pages=[int(p)], values=False)
    m, room = Model(c), Room(be)
    dev = c.put(room)
    d_slots = ints(room, slots)
    be.paged_extend(dev, d_slots, n)
    m.extend(slots, [1] * n)
    equal(c, room, dev)
    be.paged_compact(dev)
    m.compact()
    equal(c, room, dev)
    left = [s for s in range(seqs) if c.len[s] == 0][:1023]
    one = int(slots[0])
    if left and (c.refs <= 0).sum() >= len(left):
        be.paged_fork(dev, ints(room, [one] * len(left)), ints(room, left), len(left))
        m.fork([one] * len(left), left)
        equal(c, room, dev)
    room.close()


def test_the_last_page_can_be_had(be):
    c = Cache(1, pages=5, kv_heads=1, d=64, seqs=3, blocks=5)
    room = Room(be)
    dev = c.put(room)
    s = ints(room, [1])
    be.paged_extend(dev, s, 1, cu=ints(room, [0, 5 * 64]))
    assert be.paged_work(dev) == {"first": 0, "copies": 0, "live": 0, "status": 0}
    assert sorted(c.get(room, dev, "table")[0][1]) == [0, 1, 2, 3, 4]
    room.close()


def broken(be, c, call, status):
    """The call reports `status` and changes nothing but work."""
    room = Room(be)
    dev = c.put(room)
    call(be, dev, room)
    assert be.paged_work(dev)["status"] == status and be.paged_work(dev)["first"] == status
    for name, got in zip(("table", "len", "refs", "k", "v"), c.get(room, dev, "table", "len", "refs", "k", "v")):
        np.testing.assert_array_equal(got, getattr(c, name), err_msg=name)
    # the first status stays until it is cleared
    be.paged_extend(dev, ints(room, [3]), 1, cu=ints(room, [0, 0]))
    w = be.paged_work(dev)
    assert w["first"] == status and w["status"] == 0
    room.close()


def full(**kw):
    c = Cache(2, layers=2, pages=8, kv_heads=2, d=64, seqs=5, blocks=4)
    c.give(0, 100)
    c.give(1, 64)
    c.give(2, 130)
    for k, (at, v) in kw.items():
        getattr(c, k)[at] = v
    return c


A, CAP, ST = N.HYMT_E_ARG, N.HYMT_E_CAPACITY, N.HYMT_E_STATE


@pytest.mark.parametrize("slots,add,kw,status", [
    ([0, 5], [1, 1], {}, A), ([0, -1], [1, 1], {}, A), ([0, 1, 0], [1, 1, 0], {}, A), ([0, 1], [5, -2], {}, A),
    ([1, 0], [64, 200], {}, CAP),                 # more than blocks * 64 positions
    ([0, 1, 3], [29, 65, 64], {}, CAP),           # four pages, two free
    ([0], [2 ** 30], {}, CAP),
    ([0, 1, 2], [2 ** 30, 2 ** 30, 2 ** 30], {}, A),  # offsets past 2^31
    ([0], [1], {"len": (0, 257)}, ST), ([0], [1], {"len": (0, -1)}, ST),
    ([0], [1], {"table": ((0, 1), 8)}, ST), ([0], [1], {"table": ((0, 1), -1)}, ST),
])
def test_extend_that_cannot(be, slots, add, kw, status):
    broken(be, full(**kw), lambda b, dev, room: b.paged_extend(dev, ints(room, slots), len(slots),
                                                               cu=ints(room, offsets_of(add))), status)


def test_extend_of_a_shared_page(be):
    c = full()
    c.refs[c.table[0, 1]] = 2
    broken(be, c, lambda b, dev, room: b.paged_extend(dev, ints(room, [0]), 1), ST)


def test_extend_from_rows_that_do_not_begin_at_0(be):
    broken(be, full(), lambda b, dev, room: b.paged_extend(dev, ints(room, [0]), 1, cu=ints(room, [3, 4])), A)


@pytest.mark.parametrize("parent,child,kw,status", [
    ([0], [5], {}, A), ([5], [3], {}, A), ([-1], [3], {}, A), ([0, 1], [3, 3], {}, A), ([0, 3], [3, 4], {}, A),
    ([0], [1], {}, ST), ([0], [0], {}, A), ([0], [3], {"len": (0, 999)}, ST), ([0], [3], {"table": ((0, 0), 9)}, ST),
    ([0], [3], {"table": ((0, 1), -7)}, ST), ([0, 2], [3, 4], {"refs": (slice(None), 1)}, CAP),
])
def test_fork_that_cannot(be, parent, child, kw, status):
    broken(be, full(**kw), lambda b, dev, room: b.paged_fork(dev, ints(room, parent), ints(room, child), len(parent)),
           status)


@pytest.mark.parametrize("slots,lens,kw,status", [
    ([0, 5], [1, 1], {}, A), ([0, 1, 0], [1, 1, 0], {}, A), ([0, 1], [5, -2], {}, A), ([-3], [0], {}, A),
    ([0], [1], {"len": (0, 300)}, ST), ([0], [10], {"table": ((0, 0), 8)}, ST), ([2], [0], {"table": ((2, 1), -2)}, ST),
    ([2], [70], {"refs": (slice(None), 2)}, CAP),
])
def test_set_len_that_cannot(be, slots, lens, kw, status):
    broken(be, full(**kw), lambda b, dev, room: b.paged_set_len(dev, ints(room, slots), len(slots),
                                                                lens=ints(room, lens)), status)


def test_no_entries(be):
    c = full()
    room = Room(be)
    dev = c.put(room)
    s = ints(room, [9])
    be.paged_extend(dev, s, 0)
    be.paged_fork(dev, s, s, 0)
    be.paged_set_len(dev, s, 0)
    equal(c, room, dev)
    room.close()


def test_a_million_pages_for_one_slot(be):
    need = (1 << 20) + 7
    dev = be.paged_create(1, 2 * need + 3, 2, need + 1, kv_heads=1, head_dim=64)
    room = Room(be)
    try:
        be.paged_extend(dev, ints(room, [1, 0]), 2, cu=ints(room, [0, 64 * need, 64 * need + 64 * need - 63]))
        assert be.paged_work(dev) == {"first": 0, "copies": 0, "live": 0, "status": 0}
        table = be.download(np.empty((2, need + 1), np.int32), dev.table)
        refs = be.download(np.empty(2 * need + 3, np.int32), dev.refs)
        np.testing.assert_array_equal(table, [[*range(need, 2 * need), -1], [*range(need), -1]])
        np.testing.assert_array_equal(refs, [1] * (2 * need) + [0] * 3)
        be.paged_set_len(dev, ints(room, [1]), 1)
        be.paged_compact(dev)
        table = be.download(np.empty((2, need + 1), np.int32), dev.table)
        assert sorted(table[0, :need]) == [*range(need)] and (table[1] == -1).all()
    finally:
        room.close()
        be.paged_free(dev)


def test_pools_past_2_32_bytes(be):
    """Copies between pages 5 GB apart, in the last layer too."""
    pages, layers, hkv, d = 20, 1700, 8, 128
    be_cache = be.paged_create(layers, pages, 3, 4, kv_heads=hkv, head_dim=d)
    try:
        page = hkv * PAGE * d
        rng = np.random.default_rng(0)
        last = (layers - 1) * pages * page * 2
        x = rng.integers(0, 1 << 16, page, dtype=np.uint16)
        slots = Room(be)
        be.paged_extend(be_cache, ints(slots, [0]), 1, cu=ints(slots, [0, 10]))
        for pool in (be_cache.k, be_cache.v):
            be.upload(pool + last, x)
        be.paged_fork(be_cache, ints(slots, [0]), ints(slots, [2]), 1)
        for pool in (be_cache.k, be_cache.v):
            got = be.download(np.empty(page, np.uint16), pool + last + page * 2)
            np.testing.assert_array_equal(got, x)
        assert last > 1 << 32
        slots.close()
    finally:
        be.paged_free(be_cache)
