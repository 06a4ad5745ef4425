"""Steps that run out of pages: what is enqueued behind the extend that was refused
stores nothing, so the sequences are as they were, shared pages too, and the step can be
taken again once there is room (include/hymt_hip.h)."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend, Rope, rope_freqs
from hymt2sharp_amd import _native as N
from tests.paged_cases import PAGE, TINY, U, Cache, Room, batch, blocks_of, from_bits, rotated, to_bits
from tests.test_gpu_paged_pages import Model, equal, ints, offsets_of

pytestmark = pytest.mark.gpu

HEADS, HKV, D, EPS = 4, 2, 64, 1e-6


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def full(dt):
    """Slots 0 and 1 of one whole page that both hold, 2 of 70 positions; no page free."""
    c = Cache(7, layers=2, pages=3, kv_heads=HKV, d=D, dt=dt, seqs=4, blocks=70)
    c.give(0, PAGE)
    c.give(1, PAGE, pages=[int(c.table[0, 0])], values=False)
    c.give(2, 70)
    return c


def append(be, room, c, dev, layer, slots, add, pad):
    """One append, its q rows checked: its rows, and the positions and slots they are of."""
    rng = np.random.default_rng(3)
    cu = offsets_of(add)
    rows = int(cu[-1]) + pad
    x = rng.standard_normal((rows, HEADS + 2 * HKV, D)).astype(np.float32)
    px, wide = room.put(x), (HEADS + 2 * HKV) * D
    freq, scale = rope_freqs(D)
    rope = Rope(freq=room.put(freq), dim=D, interleaved=0, scale=scale)
    q0 = np.full((rows, HEADS * D), 0x1234, np.uint16)
    q = room.put(q0)
    b = batch(room, slots, cu if pad or any(a != 1 for a in add) else None, rows=rows)
    be.rope_append(dev, layer, b, px, wide, px + 4 * HEADS * D, px + 4 * (HEADS + HKV) * D, wide, N.F32, HEADS, rope, None,
                   None, EPS, q)
    pos = np.concatenate([np.arange(c.len[s] - a, c.len[s]) for s, a in zip(slots, add)])
    got = from_bits(room.get(q, q0), c.dt)[:len(pos)]
    want, err = rotated(x[:len(pos), :HEADS], pos, freq, scale, D, 0, None, EPS)
    want, err = want.reshape(len(pos), -1), err.reshape(len(pos), -1)
    assert (np.abs(got - want) <= U[c.dt] * np.abs(want) + err * 1.01 + TINY[c.dt]).all()
    return x, pos, np.repeat(slots, add), freq, scale


def stored(be, room, c, dev, layers, x, pos, of, freq, scale):
    """The rows stand in the pages of these layers, and nothing else has changed."""
    gk, gv = c.get(room, dev, "k", "v")
    want, err = rotated(x[:len(pos), HEADS:HEADS + HKV], pos, freq, scale, D, 0, None, EPS)
    for i, (s, p) in enumerate(zip(of, pos)):
        page, t = c.table[s, p // PAGE], p % PAGE
        for layer in layers:
            k = from_bits(gk[layer, page][:, c.ko[t]], c.dt)
            assert (np.abs(k - want[i]) <= U[c.dt] * np.abs(want[i]) + err[i] * 1.01 + TINY[c.dt]).all()
            c.k[layer, page][:, c.ko[t]] = gk[layer, page][:, c.ko[t]]
            c.v[layer, page][:, c.vo[t]] = to_bits(x[i, HEADS + HKV:], c.dt)
    np.testing.assert_array_equal(gk, c.k)
    np.testing.assert_array_equal(gv, c.v)


@pytest.mark.parametrize("slots,add", [([0], [1]), ([2, 0, 1], [1, 1, 1]), ([1, 2], [2, 40]), ([0, 2], [64, 3])])
@pytest.mark.parametrize("pad", [0, 1600])  # row by row, and by blocks of positions
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_rows_behind_a_refused_extend(be, slots, add, pad, dt):
    c = full(dt)
    m, room = Model(c), Room(be)
    dev = c.put(room)
    d_slots, d_cu = ints(room, slots), ints(room, offsets_of(add))
    be.paged_extend(dev, d_slots, len(slots), cu=d_cu)
    for layer in range(c.layers):
        append(be, room, c, dev, layer, slots, add, pad)
    m.end(N.HYMT_E_CAPACITY)
    equal(c, room, dev)
    # a slot that the step does not need ends; again, if that is room enough
    gone = next(s for s in (2, 1, 0) if s not in slots) if len(slots) < 3 else 2
    be.paged_set_len(dev, ints(room, [gone]), 1)
    m.set_len([gone], [0])
    equal(c, room, dev)
    keep = [(s, a) for s, a in zip(slots, add) if s != gone]
    slots, add = [s for s, _ in keep], [a for _, a in keep]
    need = sum(blocks_of(int(c.len[s]) + a) - blocks_of(int(c.len[s])) for s, a in keep)
    if need <= (c.refs == 0).sum():
        be.paged_extend(dev, ints(room, slots), len(slots), cu=ints(room, offsets_of(add)))
        m.extend(slots, add)
        for layer in range(c.layers):
            stored(be, room, c, dev, [layer], *append(be, room, c, dev, layer, slots, add, pad))
        equal(c, room, dev)
    room.close()


def test_rows_behind_any_refused_call(be):
    """While work[3] holds a status nothing is stored; the caller's clearing ends that too."""
    c = full(N.F16)
    m, room = Model(c), Room(be)
    dev = c.put(room)
    be.paged_fork(dev, ints(room, [0]), ints(room, [2]), 1)
    append(be, room, c, dev, 1, [2], [1], 0)
    m.end(N.HYMT_E_STATE)
    equal(c, room, dev)
    be.upload(dev.work, np.zeros(4, np.int32))
    c.work[:4] = 0
    stored(be, room, c, dev, [1], *append(be, room, c, dev, 1, [2], [1], 0))
    equal(c, room, dev)
    room.close()


def test_a_recorded_step_that_runs_out_of_pages(be):
    """A step recorded once and replayed: the replay that finds no page changes nothing,
    and the one after a slot has ended goes on where it stopped."""
    c = full(N.BF16)
    room = Room(be)
    dev = c.put(room)
    slots, n = ints(room, [0, 2]), 2
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, HEADS + 2 * HKV, D)).astype(np.float32)
    px, wide = room.put(x), (HEADS + 2 * HKV) * D
    freq, scale = rope_freqs(D)
    rope = Rope(freq=room.put(freq), dim=D, interleaved=0, scale=scale)
    q, out = (room.put(np.zeros((n, HEADS * D), np.uint16)) for _ in range(2))
    b = N.SeqBatch(slots=slots, n=n, rows=n, max_len=200)

    def step():
        be.paged_extend(dev, slots, n)
        for layer in range(c.layers):
            be.rope_append(dev, layer, b, px, wide, px + 4 * HEADS * D, px + 4 * (HEADS + HKV) * D, wide, N.F32, HEADS, rope,
                           None, None, EPS, q)
            be.attn_shared(dev, layer, b, 64, q, HEADS, out)

    m = Model(c)
    step()  # eagerly once, refused as well
    m.end(N.HYMT_E_CAPACITY)
    equal(c, room, dev)
    be.graph_begin()
    step()
    g = be.graph_end()
    for _ in range(3):
        be.graph_launch(g)
        be.sync()
        equal(c, room, dev)
    be.paged_set_len(dev, ints(room, [2]), 1, lens=ints(room, [60]))
    m.set_len([2], [60])
    for more in range(1, 4):
        be.graph_launch(g)
        be.sync()
        m.extend([0, 2], [1, 1])
        stored(be, room, c, dev, range(c.layers), x, np.array([c.len[0] - 1, c.len[2] - 1]), [0, 2],
               freq, scale)
        equal(c, room, dev)
    assert c.len[0] == 67 and c.len[2] == 63 and c.refs[c.table[1, 0]] == 2
    be.graph_destroy(g)
    room.close()
