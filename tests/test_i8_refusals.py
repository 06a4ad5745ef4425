"""What the 8-bit integer operators refuse, on a context without a device: the
arguments are checked before the device, so every refusal shows without a GPU
and a call that passes the checks ends in HYMT_E_NO_DEVICE.  The pointers are
addresses only and are never dereferenced."""
import ctypes

import pytest

from hymt2sharp_amd import _native as N

OK = 1 << 20


@pytest.fixture
def ctx():
    L = N.lib()
    h = ctypes.c_void_p()
    N.check(L.hymt_create(N.DEVICE_NONE, ctypes.byref(h)))
    yield L, h
    L.hymt_destroy(h)


def to_i8(L, h, x=OK, dt=N.F32, m=3, n=2048, out=OK, s=OK):
    return L.hymt_to_i8(h, x, dt, m, n, out, s)


def norm(L, h, x=OK, add=None, dt=N.BF16, m=3, n=2048, w=OK, eps=1e-6, out=OK, s=OK):
    return L.hymt_rows_rmsnorm_i8(h, x, add, dt, m, n, w, eps, out, s)


def gemm(L, h, w=OK, ws=OK, n=100, k=2048, x=OK, xs=OK, m=3, y=OK, ldy=100, flags=0):
    return L.hymt_gemm_i8(h, w, ws, n, k, x, xs, m, y, ldy, flags)


def glu(L, h, w=OK, ws=OK, up=OK, us=OK, f=100, k=2048, x=OK, xs=OK, m=3, y=OK, ld=100):
    return L.hymt_gemm_i8_swiglu(h, w, ws, up, us, f, k, x, xs, m, y, ld)


CALLS = {"to_i8": to_i8, "norm": norm, "gemm": gemm, "glu": glu}


@pytest.mark.parametrize("name", CALLS)
def test_a_good_call_reaches_the_device_check(ctx, name):
    assert CALLS[name](*ctx) == N.HYMT_E_NO_DEVICE
    assert CALLS[name](*ctx, m=0) == N.HYMT_E_NO_DEVICE
    assert CALLS[name](ctx[0], None) == N.HYMT_E_ARG
    assert CALLS[name](*ctx, m=-1) == N.HYMT_E_ARG


@pytest.mark.parametrize("name,args", [
    ("to_i8", ("x", "out", "s")), ("norm", ("x", "w", "out", "s")), ("gemm", ("w", "ws", "x", "xs", "y")),
    ("glu", ("w", "ws", "up", "us", "x", "xs", "y"))])
def test_null_pointers(ctx, name, args):
    for a in args:
        assert CALLS[name](*ctx, **{a: None}) == N.HYMT_E_ARG, a


@pytest.mark.parametrize("name,arg,bad,good", [
    ("to_i8", "x", 8, 16), ("to_i8", "out", 2, 4), ("to_i8", "s", 2, 4),
    ("norm", "x", 8, 16), ("norm", "w", 8, 16), ("norm", "add", 4, 8), ("norm", "out", 2, 4), ("norm", "s", 2, 4),
    ("gemm", "w", 8, 16), ("gemm", "x", 8, 16), ("gemm", "ws", 2, 4), ("gemm", "xs", 2, 4), ("gemm", "y", 2, 4),
    ("glu", "w", 8, 16), ("glu", "up", 8, 16), ("glu", "x", 8, 16), ("glu", "ws", 2, 4), ("glu", "us", 2, 4),
    ("glu", "xs", 2, 4), ("glu", "y", 1, 2)])
def test_alignment(ctx, name, arg, bad, good):
    assert CALLS[name](*ctx, **{arg: OK + bad}) == N.HYMT_E_ARG
    assert b"aligned" in ctx[0].hymt_last_error()
    assert CALLS[name](*ctx, **{arg: OK + good}) == N.HYMT_E_NO_DEVICE


def test_types_and_their_alignment(ctx):
    assert to_i8(*ctx, dt=N.F16) == N.HYMT_E_UNSUPPORTED
    assert to_i8(*ctx, dt=N.BF16, x=OK + 8) == N.HYMT_E_NO_DEVICE
    assert to_i8(*ctx, dt=N.BF16, x=OK + 4) == N.HYMT_E_ARG
    assert norm(*ctx, add=OK, dt=N.F16) == N.HYMT_E_UNSUPPORTED
    assert norm(*ctx, add=None, dt=N.F16) == N.HYMT_E_NO_DEVICE  # nothing to add: no type
    assert norm(*ctx, add=OK + 8, dt=N.F32) == N.HYMT_E_ARG
    assert gemm(*ctx, y=OK + 2, flags=N.GEMM_OUT_BF16) == N.HYMT_E_NO_DEVICE
    assert gemm(*ctx, y=OK + 1, flags=N.GEMM_OUT_BF16) == N.HYMT_E_ARG


@pytest.mark.parametrize("n", [0, -4, 2, 6, 2047, 8196, 1 << 30])
def test_row_lengths(ctx, n):
    assert to_i8(*ctx, n=n) == N.HYMT_E_UNSUPPORTED
    assert norm(*ctx, n=n) == N.HYMT_E_UNSUPPORTED


@pytest.mark.parametrize("k", [0, -128, 128, 64, 2000, 65536 + 128, 1 << 30])
def test_product_lengths(ctx, k):
    assert gemm(*ctx, k=k) == N.HYMT_E_UNSUPPORTED
    assert glu(*ctx, k=k) == N.HYMT_E_UNSUPPORTED


def test_sizes_and_flags(ctx):
    for bad in (dict(n=0), dict(n=-1), dict(n=101), dict(ldy=99), dict(ldy=0), dict(flags=4), dict(flags=-1),
                dict(flags=N.GEMM_ACCUMULATE | N.GEMM_OUT_BF16)):
        assert gemm(*ctx, **bad) == N.HYMT_E_ARG, bad
    for good in (dict(n=1, ldy=1), dict(ldy=101), dict(k=256), dict(k=65536), dict(m=1 << 30)):
        assert gemm(*ctx, **good) == N.HYMT_E_NO_DEVICE, good
    assert glu(*ctx, f=0) == N.HYMT_E_ARG
    assert glu(*ctx, ld=99) == N.HYMT_E_ARG
    assert norm(*ctx, eps=-1e-6) == N.HYMT_E_ARG
    assert norm(*ctx, eps=float("nan")) == N.HYMT_E_ARG
    assert norm(*ctx, eps=0.0) == N.HYMT_E_NO_DEVICE


def test_weight_codes_need_a_weight(ctx):
    L, h = ctx
    a, b = ctypes.c_void_p(), ctypes.c_void_p()
    assert L.hymt_weight_i8(h, None) == N.HYMT_E_NO_DEVICE
    assert L.hymt_weight_i8(None, None) == N.HYMT_E_ARG
    assert L.hymt_weight_i8_data(None, ctypes.byref(a), ctypes.byref(b)) == N.HYMT_E_ARG
