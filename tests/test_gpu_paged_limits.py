"""The attention over the multi-sequence cache at the ends of what its entry points
accept."""
import contextlib

import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import Cache
from tests.test_gpu_paged_attn import run, cu_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


@contextlib.contextmanager
def launches(be):
    """Launches of the two kernels within."""
    n = {}
    be.timing_enable(2)
    be.timing_reset()
    yield n
    for k in ("attn_shared", "attn_merge"):
        try:
            n[k] = be.timing(k)[0]
        except ValueError:  # never timed
            n[k] = 0
    be.timing_enable(0)


def test_rows_of_sequences_that_could_have_2_24_pages(be):
    """1024 rows of 32 kv heads fill the chip: nothing is cut, however long the slots
    could be."""
    c = Cache(1, pages=2, kv_heads=32, d=64, dt=N.F16, seqs=1, blocks=1 << 24)
    c.give(0, 70)
    with launches(be) as n:
        run(be, c, [0] * 1024, None, 32, prefix=0)
    assert n == {"attn_shared": 1, "attn_merge": 0}


@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127])
@pytest.mark.parametrize("new,lens,prefix", [([70, 9], [70, 200], None), ([20], [3000], None), ([1, 1], [70, 200], 0),
                                             ([1, 1], [70, 2000], 64)])
def test_the_largest_scale(be, scale, new, lens, prefix):
    """Scores of 0 times the largest scale are 0: the mean of V."""
    c = Cache(2, pages=60, kv_heads=1, d=64, dt=N.BF16, seqs=2, blocks=50)
    for i, n in enumerate(lens):
        c.give(i, n)
    if prefix:
        c.table[1, 0] = c.table[0, 0]
    run(be, c, [0, 1][:len(new)], None if prefix is not None else cu_of(new), 4, scale=scale, prefix=prefix,
        q=np.zeros((sum(new), 4 * 64)))


@pytest.mark.parametrize("length,merges", [(8192, 0), (8300, 1)])
@pytest.mark.parametrize("dt", [N.F16, N.BF16])
def test_long_ranges_of_rows_for_half_of_the_chip(be, length, merges, dt):
    """32 rows of 4 kv heads: whole up to 128 pages, cut in two beyond."""
    c = Cache(4, pages=131, kv_heads=4, d=64, dt=dt, seqs=2, blocks=140)
    c.give(1, length)
    with launches(be) as n:
        run(be, c, [1] * 32, None, 8, prefix=0, max_len=length)
    assert n == {"attn_shared": 1, "attn_merge": merges}
