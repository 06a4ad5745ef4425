"""An allocation that finds no room is refused with HYMT_E_OOM, and the calls
after it are none the worse."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from tests.i8_cases import Room, codes_of

pytestmark = pytest.mark.gpu


def test_calls_after_a_refused_allocation(hip_available):
    be = HipBackend(0)
    try:
        x = np.random.default_rng(1).standard_normal((3, 512)).astype(np.float32)
        r = Room(be)
        dx, dg = r.put(x), r.put(np.ones(512, np.float32))
        dq, ds = r.put(np.zeros((3, 512), np.int8)), r.put(np.zeros(3, np.float32))
        db = r.put(np.zeros((3, 512), np.uint16))
        calls = [lambda: be.to_i8(dx, 3, 512, dq, ds),
                 lambda: be.rows_rmsnorm_i8(dx, 3, 512, dg, 1e-5, dq, ds),
                 lambda: be.gemm_i8(dq, ds, 3, 512, dq, ds, 3, db, out_bf16=True),
                 lambda: be.to_bf16(dx, 1536, db)]
        for call in calls:
            with pytest.raises(MemoryError):
                be.alloc(1 << 46)
            call()
        be.to_i8(dx, 3, 512, dq, ds)
        np.testing.assert_array_equal(r.get(dq, np.empty((3, 512), np.int8)), codes_of(x)[0])
        r.close()
    finally:
        be.Dispose()
