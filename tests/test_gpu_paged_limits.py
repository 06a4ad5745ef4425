"""The attention over the multi-sequence cache at the ends of what its entry points
accept."""
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from tests.paged_cases import Cache
from tests.test_gpu_paged_attn import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = HipBackend(0)
    yield b
    b.Dispose()


def test_rows_of_sequences_that_could_have_2_24_pages(be):
    """1024 rows of 32 kv heads fill the chip: nothing is cut, however long the slots
    could be."""
    c = Cache(1, pages=2, kv_heads=32, d=64, dt=N.F16, seqs=1, blocks=1 << 24)
    c.give(0, 70)
    be.timing_enable(2)
    be.timing_reset()
    run(be, c, [0] * 1024, None, 32, prefix=0)
    calls, merges = be.timing("attn_shared")[0], 0
    try:
        merges = be.timing("attn_merge")[0]
    except ValueError:
        pass
    be.timing_enable(0)
    assert calls == 1 and merges == 0
