"""HYMT_HIP_I8_TILE on a context without a device: the names of the tiles pass
and reach the device check, any other is refused by both products."""
import ctypes

import pytest

from hymt2sharp_amd import _native as N
from tests.test_gpu_i8_gemm import TILES
from tests.test_i8_refusals import gemm, glu


@pytest.fixture
def ctx():
    L = N.lib()
    h = ctypes.c_void_p()
    N.check(L.hymt_create(N.DEVICE_NONE, ctypes.byref(h)))
    yield L, h
    L.hymt_destroy(h)


@pytest.mark.parametrize("tile", TILES)
def test_the_tiles_that_the_tests_name(ctx, monkeypatch, tile):
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    assert gemm(*ctx) == N.HYMT_E_NO_DEVICE
    assert glu(*ctx) == N.HYMT_E_NO_DEVICE


@pytest.mark.parametrize("tile", ["", "64", "64x48", "64X64", "64x64 ", "256x2561", "128x64,2"])
def test_any_other_name_is_refused(ctx, monkeypatch, tile):
    monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
    for call in (gemm, glu):
        assert call(*ctx) == N.HYMT_E_ARG
        assert b"HYMT_HIP_I8_TILE" in ctx[0].hymt_last_error()
    monkeypatch.delenv("HYMT_HIP_I8_TILE")
    assert gemm(*ctx) == N.HYMT_E_NO_DEVICE
