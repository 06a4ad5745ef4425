"""The multi-sequence cache's operators together, as a server uses them: an
instruction's prompt, forks of it, their own prompts packed, steps of single
tokens, ends, a compacted pool, and steps again -- checked after every call --
and a step recorded once and replayed as the sequences grow."""
import ctypes

import numpy as np
import pytest

from hymt2sharp_amd import HipBackend, Rope, rope_freqs
from hymt2sharp_amd import _native as N
from tests.i8_cases import Room
from tests.paged_cases import PAGE, TINY, U, Cache, attention, batch, blocks_of, check_rows, from_bits, rotated, to_bits
from tests.test_gpu_paged_pages import Model, equal, ints, offsets_of

pytestmark = pytest.mark.gpu

HEADS, HKV, D, LAYERS = 8, 2, 64, 2
EPS = 1e-6


class Server:
    def __init__(self, be, dt, seed=0):
        self.be, self.room, self.rng = be, Room(be), np.random.default_rng(seed)
        self.c = Cache(seed, layers=LAYERS, pages=60, kv_heads=HKV, d=D, dt=dt, seqs=10, blocks=12)
        self.m = Model(self.c)
        self.dev = self.c.put(self.room)
        self.freq, self.scale = rope_freqs(D, 10000.0, N.ROPE_YARN, 4.0, 256)
        self.rope = Rope(freq=self.room.put(self.freq), dim=D, interleaved=0, scale=self.scale)
        self.w = [self.rng.uniform(0.8, 1.2, D).astype(np.float32) for _ in range(2)]
        self.dw = [self.room.put(x) for x in self.w]

    def close(self):
        assert self.be.paged_work(self.dev)["first"] == 0
        self.room.close()

    def extend(self, slots, add):
        self.be.paged_extend(self.dev, ints(self.room, slots), len(slots), cu=ints(self.room, offsets_of(add)))
        self.m.extend(slots, add)
        equal(self.c, self.room, self.dev)

    def layer(self, layer, slots, add, prefix=None):
        """Append and attend in one layer, each against its reference over the
        cache as it stands."""
        c, room, cu = self.c, self.room, offsets_of(add).tolist()
        rows, dt = cu[-1], c.dt
        x = self.rng.standard_normal((rows, HEADS + 2 * HKV, D)).astype(np.float32)
        xq, xk, xv = (room.put(x[:, a:b].reshape(rows, -1)) for a, b in ((0, HEADS), (HEADS, HEADS + HKV),
                                                                         (HEADS + HKV, HEADS + 2 * HKV)))
        one = all(a == 1 for a in add)
        b = batch(room, slots, None if one else cu, rows=rows, max_len=int(c.len.max()))
        q = room.put(np.zeros((rows, HEADS * D), np.uint16))
        self.be.rope_append(self.dev, layer, b, xq, HEADS * D, xk, xv, HKV * D, N.F32, HEADS, self.rope, *self.dw, EPS, q)
        gq = room.get(q, np.zeros((rows, HEADS * D), np.uint16))
        gk, gv = c.get(room, self.dev, "k", "v")
        pos = np.concatenate([np.arange(c.len[s] - a, c.len[s]) for s, a in zip(slots, add)])
        of = np.repeat(slots, add)

        def near(got, want, err):
            assert (np.abs(from_bits(got, dt) - want) <= U[dt] * np.abs(want) + err * 1.01 + TINY[dt]).all()

        y, err = rotated(x[:, :HEADS], pos, self.freq, self.scale, D, 0, self.w[0], EPS)
        near(gq, y.reshape(rows, -1), err.reshape(rows, -1))
        y, err = rotated(x[:, HEADS:HEADS + HKV], pos, self.freq, self.scale, D, 0, self.w[1], EPS)
        for i in range(rows):
            p, t = c.table[of[i], pos[i] // PAGE], pos[i] % PAGE
            near(gk[layer, p][:, c.ko[t]], y[i], err[i])
            c.k[layer, p][:, c.ko[t]] = gk[layer, p][:, c.ko[t]]
            c.v[layer, p][:, c.vo[t]] = to_bits(x[i, HEADS + HKV:], dt)
        np.testing.assert_array_equal(gk, c.k)
        np.testing.assert_array_equal(gv, c.v)
        before = np.full((rows, HEADS * D), 0x3C3C, np.uint16)
        out = room.put(before)
        if prefix is None:
            self.be.attn_packed(self.dev, layer, b, q, HEADS, out)
        else:
            self.be.attn_shared(self.dev, layer, b, prefix, q, HEADS, out)
        want, tol, done = attention(c, layer, slots, None if one else cu, from_bits(gq, dt), HEADS, prefix=prefix or 0)
        check_rows(room.get(out, before), want, tol, done, before, dt)

    def rows(self, slots, add, prefix=None):
        self.extend(slots, add)
        for layer in range(LAYERS):
            self.layer(layer, slots, add, prefix)


@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_a_server(be, dt):
    s = Server(be, dt)
    s.rows([4], [150])                               # the instruction
    be.paged_fork(s.dev, ints(s.room, [4] * 4), ints(s.room, [0, 9, 2, 7]), 4)
    s.m.fork([4] * 4, [0, 9, 2, 7])
    equal(s.c, s.room, s.dev)
    s.rows([9, 0, 7, 2], [30, 1, 106, 0])            # the requests
    for _ in range(3):
        s.rows([0, 2, 7, 9], [1] * 4, prefix=128)    # tokens
    s.rows([0, 2, 7, 9], [2, 1, 3, 1])               # tokens and drafts
    be.paged_set_len(s.dev, ints(s.room, [7, 0]), 2, lens=ints(s.room, [257, 100]))  # drafts that were wrong
    s.m.set_len([7, 0], [257, 100])
    equal(s.c, s.room, s.dev)
    be.paged_set_len(s.dev, ints(s.room, [4, 9]), 2)  # the instruction's slot and a request end
    s.m.set_len([4, 9], [0, 0])
    equal(s.c, s.room, s.dev)
    be.paged_compact(s.dev)
    s.m.compact()
    equal(s.c, s.room, s.dev)
    s.rows([2, 7], [1, 1], prefix=128)
    s.rows([4, 0], [65, 3])                          # a new request beside an old one
    s.rows([0, 2, 4, 7], [1] * 4, prefix=0)
    s.close()


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def step_of(be, dev, slots, n, prefix, rope, x, q, out, max_len):
    """One token of every slot, enqueued: the positions come from the cache."""
    b = N.SeqBatch(slots=slots, n=n, rows=n, max_len=max_len)
    be.paged_extend(dev, slots, n)
    for layer in range(LAYERS):
        wide = (HEADS + 2 * HKV) * D
        be.rope_append(dev, layer, b, x, wide, x + 4 * HEADS * D, x + 4 * (HEADS + HKV) * D, wide, N.F32, HEADS, rope, None,
                       None, EPS, q)
        be.attn_shared(dev, layer, b, prefix, q, HEADS, out + 2 * layer * n * HEADS * D)


@pytest.mark.parametrize("prefix,most", [(0, 600), (192, 600), (192, 2500)])
def test_a_recorded_step_follows_the_lengths(be, prefix, most):
    """Two equal caches, one stepped by replays, one eagerly, compared bit by bit
    after every step, over a page's end and with other work between the replays."""
    rng = np.random.default_rng(1)
    n, slots = 5, [3, 0, 4, 1, 2]
    sides = []
    room = Room(be)
    freq, scale = rope_freqs(D)
    rope = Rope(freq=room.put(freq), dim=D, interleaved=1, scale=scale)
    for _ in range(2):
        c = Cache(4, layers=LAYERS, pages=70, kv_heads=HKV, d=D, dt=N.BF16, seqs=6, blocks=40)
        for i, s in enumerate(slots):
            pages = None if i == 0 or not prefix else c.table[slots[0], :prefix // PAGE].tolist() + [
                int(p) for p in np.flatnonzero(c.refs == 0)]
            c.give(s, prefix + [61, 1, 64, 30, 300][i], pages=pages)
        sides.append([c, c.put(room)])
    np.testing.assert_array_equal(sides[0][0].k, sides[1][0].k)
    x = room.put(rng.standard_normal((n, HEADS + 2 * HKV, D)).astype(np.float32))
    d_slots = ints(room, slots)
    q = room.put(np.zeros((n, HEADS * D), np.uint16))
    outs = [room.put(np.zeros((LAYERS, n, HEADS * D), np.uint16)) for _ in range(2)]
    args = lambda k: (be, sides[k][1], d_slots, n, prefix, rope, x, q, outs[k], most)
    step_of(*args(0))  # workspaces grow outside the recording
    step_of(*args(1))
    be.graph_begin()
    step_of(*args(0))
    g = be.graph_end()
    zero = np.zeros((LAYERS, n, HEADS * D), np.uint16)
    for step in range(6):
        be.graph_launch(g)
        step_of(*args(1))
        be.sync()
        a, b = (room.get(o, zero) for o in outs)
        np.testing.assert_array_equal(a, b, err_msg=str(step))
        for name, p, r in zip(("table", "len", "refs", "k", "v"), *(s[0].get(room, s[1], "table", "len", "refs", "k", "v")
                                                                     for s in sides)):
            np.testing.assert_array_equal(p, r, err_msg=f"{name} {step}")
        assert np.isfinite(from_bits(a, N.BF16)).all() and (a != 0).any()
    lens = sides[0][0].get(room, sides[0][1], "len")[0]
    assert lens[slots[0]] == prefix + 61 + 7
    be.graph_destroy(g)
    assert all(be.paged_work(s[1])["first"] == 0 for s in sides)
    room.close()


def test_a_recording_that_would_have_to_grow(be):
    """The workspace of a cut range may not grow while recording; upkeep and
    calls without one are recorded."""
    fresh = HipBackend(0)
    room = Room(fresh)
    try:
        c = Cache(1, pages=60, kv_heads=1, d=D, seqs=2, blocks=60)
        c.give(0, 3000)
        dev = c.put(room)
        q, out = (room.put(np.zeros((1, 2 * D), np.uint16)) for _ in range(2))
        b = batch(room, [0], max_len=3000)
        fresh.graph_begin()
        with pytest.raises(N.InvalidOperationError):
            fresh.attn_shared(dev, 0, b, 0, q, 2, out)
        with pytest.raises(N.InvalidOperationError):
            fresh.graph_end()
        small = batch(room, [0], max_len=64)
        fresh.graph_begin()
        fresh.attn_shared(dev, 0, small, 0, q, 2, out)
        fresh.paged_compact(dev)
        g = fresh.graph_end()
        fresh.graph_launch(g)
        fresh.graph_destroy(g)
    finally:
        room.close()
        fresh.Dispose()


def test_a_recording_whose_workspace_was_replaced(be):
    """Two recordings share the workspace and give the eager bits in any order; once
    an eager call has made it grow, they are refused."""
    fresh = HipBackend(0)
    room = Room(fresh)
    try:
        c = Cache(1, pages=300, kv_heads=1, d=D, seqs=3, blocks=200)
        c.give(0, 3000)
        c.give(1, 12000)
        dev = c.put(room)
        rng = np.random.default_rng(0)
        q = room.put(to_bits(rng.standard_normal((40, 2 * D)), N.BF16))
        zero = np.zeros((40, 2 * D), np.uint16)
        outs = [room.put(zero) for _ in range(4)]
        one = batch(room, [0], max_len=3000)
        rows = batch(room, [0], [0, 40], max_len=3000)
        calls = [lambda o: fresh.attn_shared(dev, 0, one, 0, q, 2, o), lambda o: fresh.attn_packed(dev, 0, rows, q, 2, o)]
        for f, o in zip(calls, outs):
            f(o)
        graphs = []
        for f, o in zip(calls, outs[2:]):
            fresh.graph_begin()
            f(o)
            graphs.append(fresh.graph_end())
        for order in ([0, 1, 0], [1, 1, 0], [0, 1]):
            for o in outs[2:]:
                fresh.upload(o, zero)
            for k in order:
                fresh.graph_launch(graphs[k])
            fresh.sync()
            for k in range(2):
                np.testing.assert_array_equal(room.get(outs[2 + k], zero), room.get(outs[k], zero))
        fresh.attn_packed(dev, 0, batch(room, [0, 1], [0, 1, 40], max_len=12000), q, 2, outs[0])
        for g in graphs:
            with pytest.raises(N.InvalidOperationError):
                fresh.graph_launch(g)
            fresh.graph_destroy(g)
    finally:
        room.close()
        fresh.Dispose()


@pytest.mark.parametrize("new,lens,prefix", [([70, 3], [300, 900], None), ([2000], [2000], None), ([5] * 3, [4000] * 3, None),
                                             ([1] * 5, [100, 1, 64, 700, 9], 0), ([1] * 2, [3000, 5000], 0),
                                             ([1] * 40, [700] * 40, 640), ([1] * 5, [1500] * 5, 640)])
def test_out_may_be_q(be, new, lens, prefix):
    room = Room(be)
    hkv, group = 2, 20 if prefix == 0 else 3
    c = Cache(3, pages=sum(blocks_of(n) for n in lens), kv_heads=hkv, d=D, dt=N.F16, seqs=len(lens), blocks=100)
    for i, n in enumerate(lens):
        c.give(i, n)
    if prefix:
        c.table[:, :prefix // PAGE] = c.table[0, :prefix // PAGE]
    dev = c.put(room)
    cu = None if prefix is not None else np.concatenate([[0], np.cumsum(new)])
    b = batch(room, range(len(lens)), cu, max_len=max(lens))
    bits = to_bits(np.random.default_rng(1).standard_normal((sum(new), hkv * group * D)), N.F16)
    q, x, out = room.put(bits), room.put(bits), room.put(np.zeros_like(bits))
    for source, to in ((q, out), (x, x)):
        if prefix is None:
            be.attn_packed(dev, 0, b, source, hkv * group, to)
        else:
            be.attn_shared(dev, 0, b, prefix, source, hkv * group, to)
    np.testing.assert_array_equal(room.get(x, bits), room.get(out, bits))
    np.testing.assert_array_equal(room.get(q, bits), bits)
    room.close()


@pytest.mark.parametrize("n", [5, 64, 65, 300, 1024])
def test_offsets_and_slots_that_mean_nothing(be, n):
    """Whatever slots, cu, table and len hold, nothing outside the buffers is written
    (Room.close checks their surroundings) and the calls end; the cache's lists are
    read only."""
    rng = np.random.default_rng(n)
    rows, heads, hkv, d = 700, 4, 2, 64
    for kind in ("random", "alternating", "near"):
        c = Cache(n, pages=40, kv_heads=hkv, d=d, dt=N.F16, seqs=9, blocks=5)
        c.table[:] = rng.integers(-3, 45, c.table.shape)
        c.len[:] = rng.integers(-50, 400, c.len.shape)
        c.table[0, 0], c.len[1], c.len[2] = 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31
        cu = {"random": rng.integers(-2 ** 31, 2 ** 31, n + 1), "alternating": np.arange(n + 1) % 2 * rows,
              "near": rng.integers(-5, rows + 5, n + 1)}[kind]
        slots = rng.integers(-2, 12, n)
        slots[0] = 2 ** 31 - 1
        room = Room(be)
        dev = c.put(room)
        b = batch(room, slots, cu, rows=rows, max_len=300)
        x = room.put(rng.standard_normal((rows, heads + 2 * hkv, d)).astype(np.float32))
        freq, scale = rope_freqs(d)
        rope = Rope(freq=room.put(freq), dim=d, interleaved=0, scale=scale)
        q = room.put(to_bits(rng.standard_normal((max(rows, n), heads * d)), N.F16))
        out = room.put(np.zeros((max(rows, n), heads * d), np.uint16))
        wide = (heads + 2 * hkv) * d
        be.attn_packed(dev, 0, b, q, heads, out)
        for prefix in (0, 128):
            be.attn_shared(dev, 0, batch(room, slots), prefix, q, heads, out)
        for more in (0, 1):  # row by row and by blocks
            if more:
                x = room.put(rng.standard_normal((16 * max(n, 100), wide)).astype(np.float32))
                q = room.put(np.zeros((16 * max(n, 100), heads * d), np.uint16))
                b = batch(room, slots, cu, rows=16 * max(n, 100))
            be.rope_append(dev, 0, b, x, wide, x + 4 * heads * d, x + 4 * (heads + hkv) * d, wide, N.F32, heads, rope, None,
                           None, EPS, q)
        be.sync()
        for name, got in zip(("table", "len", "refs"), c.get(room, dev, "table", "len", "refs")):
            np.testing.assert_array_equal(got, getattr(c, name), err_msg=name)
        room.close()


def test_the_most_rows(be):
    """2^22 rows in 1024 sequences of 4096 through the append and the attention: byte
    offsets past 2^31, rows looked at where blocks, tiles and sequences meet."""
    n, length, heads, hkv, d = 1024, 4096, 4, 1, 64
    rows, wide, some = n * length, (heads + 2 * hkv) * d, 4096 - 7
    rng = np.random.default_rng(0)
    x = to_bits(rng.standard_normal((some, wide)), N.F16)  # row r of the batch is x[r % some]
    room = Room(be)
    c = be.paged_create(1, n * length // PAGE, n, length // PAGE, kv_heads=hkv, head_dim=d, dtype=N.F16)
    qkv, q = be.alloc(rows * wide * 2), be.alloc(rows * heads * d * 2)
    try:
        for r in range(0, rows, some):
            part = x[:min(some, rows - r)]
            be.upload(qkv + r * wide * 2, part)
        slots = rng.permutation(n).astype(np.int32)
        d_slots, cu = ints(room, slots), ints(room, np.arange(n + 1) * length)
        b = N.SeqBatch(slots=d_slots, cu=cu, n=n, rows=rows, max_len=length)
        freq, scale = rope_freqs(d)
        rope = Rope(freq=room.put(freq), dim=d, interleaved=0, scale=scale)
        be.paged_extend(c, d_slots, n, cu=cu)
        be.rope_append(c, 0, b, qkv, wide, qkv + heads * d * 2, qkv + (heads + hkv) * d * 2, wide, N.F16, heads, rope, None,
                       None, EPS, q)
        got_q = {}
        entries = {0: [0, 1, 4095], 1: [0, 31], 511: [2047, 2048], 1022: [4064], 1023: [4063, 4064, 4095]}
        for e, some_rows in entries.items():
            for i in some_rows:
                r = e * length + i
                got_q[r] = be.download(np.empty(heads * d, np.uint16), q + r * heads * d * 2)
                y, err = rotated(from_bits(x[r % some], N.F16)[None, :heads * d].reshape(1, heads, d), np.array([i]), freq,
                                 scale, d, 0, None, EPS)
                near = np.abs(from_bits(got_q[r], N.F16) - y.reshape(-1))
                assert (near <= U[N.F16] * np.abs(y.reshape(-1)) + err.reshape(-1) * 1.001 + TINY[N.F16]).all(), r
        be.attn_packed(c, 0, b, q, heads, q)  # in place
        assert be.paged_work(c)["first"] == 0
        table = be.download(np.empty((n, length // PAGE), np.int32), c.table)
        one = Cache(0, pages=length // PAGE, kv_heads=hkv, d=d, dt=N.F16, seqs=1, blocks=length // PAGE)
        one.len[0], one.table[0] = length, np.arange(length // PAGE)
        for e, some_rows in entries.items():
            for k, page in enumerate(table[slots[e]]):
                for pool, to in ((c.k, one.k), (c.v, one.v)):
                    to[0, k, 0] = be.download(np.empty(PAGE * d, np.uint16), pool + int(page) * PAGE * d * 2)
            v = one.rows(0, 0, length)[1][0]
            np.testing.assert_array_equal(v, from_bits(x[(e * length + np.arange(length)) % some], N.F16)[:, -d:])
            for i in some_rows:
                r = e * length + i
                one.len[0] = i + 1  # the row as a sequence's last
                want, tol, done = attention(one, 0, [0], None, from_bits(got_q[r], N.F16)[None], heads)
                got = be.download(np.empty((1, heads * d), np.uint16), q + r * heads * d * 2)
                check_rows(got, want, tol, done, got, N.F16)
            one.len[0] = length
    finally:
        be.free(qkv)
        be.free(q)
        be.paged_free(c)
        room.close()


def test_kernels_are_timed(be):
    room = Room(be)
    c = Cache(1, pages=60, kv_heads=1, d=D, seqs=2, blocks=60)
    c.give(0, 2900)
    dev = c.put(room)
    q, out = (room.put(np.zeros((2, 2 * D), np.uint16)) for _ in range(2))
    be.timing_enable(2)
    be.timing_reset()
    s = ints(room, [0])
    be.paged_extend(dev, s, 1)
    be.paged_fork(dev, s, ints(room, [1]), 1)
    be.attn_shared(dev, 0, batch(room, [0, 1], max_len=2901), 64, q, 2, out)
    be.attn_packed(dev, 0, batch(room, [0, 1], [0, 1, 2], max_len=2901), q, 2, out)
    be.sync()
    for k in ("paged_extend", "paged_plan", "paged_copy", "attn_shared", "attn_packed", "attn_merge"):
        assert be.timing(k)[0] >= 1, k
    be.timing_enable(0)
    room.close()


def test_host_buffers_and_errors_of_the_mirror(be):
    c = be.paged_create(2, 8, 3, 4, kv_heads=2, head_dim=64, dtype=N.F16)
    assert be.paged_work(c) == {"first": 0, "copies": 0, "live": 0, "status": 0}
    with pytest.raises(ValueError):
        be.attn_packed(c, 2, N.SeqBatch(slots=c.len, n=1, rows=1), c.k, 4, c.v)
    with pytest.raises(N.NotSupportedError):
        be.attn_packed(c, 0, N.SeqBatch(slots=c.len, n=1, rows=1), c.k, 2 * 65, c.v)
    be.paged_free(c)
    assert c.k is None and c.work is None
    assert ctypes.sizeof(N.PagedCache) == 80 and ctypes.sizeof(N.SeqBatch) == 32 and ctypes.sizeof(N.Rope) == 24
