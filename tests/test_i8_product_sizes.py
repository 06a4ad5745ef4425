"""The largest int8 products, on a context without a device: what a launch cannot
hold is refused as such, before the device is asked."""
import ctypes

import pytest

from hymt2sharp_amd import _native as N
from tests.test_i8_refusals import gemm, glu


@pytest.fixture
def ctx():
    L = N.lib()
    h = ctypes.c_void_p()
    N.check(L.hymt_create(N.DEVICE_NONE, ctypes.byref(h)))
    yield L, h
    L.hymt_destroy(h)


@pytest.mark.parametrize("n,m,fits", [
    (256, 1 << 30, True), (257, 1 << 30, False), (257, 1 << 29, True), (257, (1 << 29) + 1, False),
    (1 << 30, 256, True), (1 << 30, 257, False), (1 << 30, 0, True)])
def test_products(ctx, n, m, fits):
    want = N.HYMT_E_NO_DEVICE if fits else N.HYMT_E_UNSUPPORTED
    for flags in (0, N.GEMM_ACCUMULATE, N.GEMM_OUT_BF16):
        assert gemm(*ctx, n=n, m=m, ldy=n, flags=flags) == want


@pytest.mark.parametrize("f,m,fits", [
    (128, 1 << 30, True), (129, 1 << 30, False), (129, 1 << 29, True), (129, (1 << 29) + 1, False),
    (1 << 29, 256, True), (1 << 29, 257, False), ((1 << 29) + 1, 256, False)])
def test_swiglu(ctx, f, m, fits):
    assert glu(*ctx, f=f, m=m, ld=f) == (N.HYMT_E_NO_DEVICE if fits else N.HYMT_E_UNSUPPORTED)
