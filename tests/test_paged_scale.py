"""Scales of the attention over the multi-sequence cache near fp32's largest number, on a
context without a device: one whose product with log2 e is no number is refused."""
import ctypes

import pytest

from hymt2sharp_amd import _native as N
from tests.test_paged_refusals import packed, shared


@pytest.fixture
def ctx():
    L = N.lib()
    h = ctypes.c_void_p()
    N.check(L.hymt_create(N.DEVICE_NONE, ctypes.byref(h)))
    yield L, h
    L.hymt_destroy(h)


@pytest.mark.parametrize("f", [packed, shared])
@pytest.mark.parametrize("sign", [1, -1])
def test_scales(ctx, f, sign):
    # fp32's largest number, 3.4028e38, over 1.442695 is 2.3587e38
    for good in (2.0 ** 127, 2.35e38, 1e-45, 0.0):
        assert f(*ctx, scale=sign * good) == N.HYMT_E_NO_DEVICE, good
    for bad in (2.37e38, 3.4028234e38, float("inf")):
        assert f(*ctx, scale=sign * bad) == N.HYMT_E_ARG, bad
    assert b"scale" in ctx[0].hymt_last_error()
