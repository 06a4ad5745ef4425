"""Reference counts that the rules of the multi-sequence cache exclude, among those that
an upkeep call goes by: it is refused and changes nothing (include/hymt_hip.h).  And
counts that the rules allow, up to large ones, which pass."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import Cache, Room
from tests.test_gpu_paged_pages import Model, broken, equal, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def held(*counts):
    """Slots 0 (130 positions), 1 (64) and 2 (10000, 157 pages); counts are (slot, block,
    count)."""
    c = Cache(3, layers=2, pages=170, kv_heads=1, d=64, seqs=6, blocks=160)
    c.give(0, 130)
    c.give(1, 64)
    c.give(2, 10000)
    for slot, block, n in counts:
        c.refs[c.table[slot, block]] = n
    return c


FORKS = [
    ([0], [4], [(0, 0, 0)]), ([0], [4], [(0, 1, 0)]), ([0], [4], [(0, 1, -1)]), ([1], [4], [(1, 0, 0)]),
    ([0], [4], [(0, 2, 0)]), ([0], [4], [(0, 2, 2)]), ([0], [4], [(0, 2, -2 ** 31)]), ([0], [4], [(0, 2, 2 ** 31 - 1)]),
    ([1, 2], [4, 5], [(2, 155, 0)]), ([1, 2], [4, 5], [(2, 64, 0)]), ([2, 1], [4, 5], [(2, 156, 0)]),
    # page 0 of slot 0 is free by its count: it could be the copy of slot 2's last one
    ([2, 0], [4, 5], [(0, 0, 0)]),
]


@pytest.mark.parametrize("parent,child,counts", FORKS)
def test_fork_of_pages_without_their_count(be, parent, child, counts):
    broken(be, held(*counts), lambda b, dev, room: b.paged_fork(dev, ints(room, parent), ints(room, child), len(parent)),
           N.HYMT_E_STATE)


CUTS = [
    ([0], [0], [(0, 0, 0)]), ([0], [0], [(0, 2, 0)]), ([0], [0], [(0, 1, -5)]), ([0], [64], [(0, 1, 0)]),
    ([0], [70], [(0, 2, 0)]), ([0], [70], [(0, 1, 0)]), ([1, 2], [64, 1], [(2, 156, 0)]), ([2, 1], [4000, 0], [(2, 100, 0)]),
    ([1, 2], [0, 9999], [(1, 0, -1)]),
]


@pytest.mark.parametrize("slots,lens,counts", CUTS)
def test_cut_of_pages_without_their_count(be, slots, lens, counts):
    broken(be, held(*counts), lambda b, dev, room: b.paged_set_len(dev, ints(room, slots), len(slots),
                                                                   lens=ints(room, lens)), N.HYMT_E_STATE)


@pytest.mark.parametrize("counts", [[(0, 0, 0)], [(0, 2, 0)], [(2, 0, -1)]])
def test_release_of_pages_without_their_count(be, counts):
    broken(be, held(*counts), lambda b, dev, room: b.paged_set_len(dev, ints(room, [1, 2, 0]), 3), N.HYMT_E_STATE)


def test_counts_that_the_calls_do_not_go_by(be):
    """Other sequences' counts, and those of pages that a cut keeps, are their own affair."""
    c = held((0, 0, 0), (1, 0, 0))
    m, room = Model(c), Room(be)
    dev = c.put(room)
    be.paged_set_len(dev, ints(room, [0, 2]), 2, lens=ints(room, [64, 9990]))
    m.set_len([0, 2], [64, 9990])
    equal(c, room, dev)
    room.close()


def test_large_counts(be):
    """Whole pages that many hold: one more, and one less."""
    c = held((0, 0, 2 ** 30), (0, 1, 65535))
    m, room = Model(c), Room(be)
    dev = c.put(room)
    be.paged_fork(dev, ints(room, [0, 0]), ints(room, [4, 5]), 2)
    m.fork([0, 0], [4, 5])
    equal(c, room, dev)
    be.paged_set_len(dev, ints(room, [0, 5]), 2, lens=ints(room, [70, 0]))
    m.set_len([0, 5], [70, 0])
    equal(c, room, dev)
    assert be.paged_work(dev) == {"first": 0, "copies": 1, "live": 0, "status": 0}
    assert np.count_nonzero(c.refs[c.table[0, :2]] > 1) == 1
    room.close()
