"""What the multi-sequence cache's entry points refuse, on a context without a
device: the arguments are checked before the device, so every refusal shows without a
GPU and a call that passes the checks ends in HYMT_E_NO_DEVICE.  The pointers are
addresses only and are never dereferenced.  And hymt_rope_freqs, which needs no
device, against its formulas."""
import ctypes
import math

import numpy as np
import pytest

from hymt2sharp_amd import ROPE_LINEAR, ROPE_NONE, ROPE_NTK, ROPE_YARN, rope_freqs
from hymt2sharp_amd import _native as N

OK = 1 << 20


@pytest.fixture
def ctx():
    L = N.lib()
    h = ctypes.c_void_p()
    N.check(L.hymt_create(N.DEVICE_NONE, ctypes.byref(h)))
    yield L, h
    L.hymt_destroy(h)


def cache(**kw):
    d = dict(k=OK, v=OK, table=OK, len=OK, refs=OK, work=OK, layers=2, pages=9, kv_heads=4, head_dim=128, dtype=N.BF16,
             seqs=5, blocks=7)
    d.update(kw)
    return N.PagedCache(**d)


def batch(**kw):
    d = dict(slots=OK, cu=OK, n=3, rows=10, max_len=0)
    d.update(kw)
    return N.SeqBatch(**d)


def rope(**kw):
    d = dict(freq=OK, dim=128, interleaved=0, scale=1.0)
    d.update(kw)
    return N.Rope(**d)


def ref(s):
    return None if s is None else ctypes.byref(s)


def extend(L, h, c=cache(), a=OK, b=OK, n=3):
    return L.hymt_paged_extend(h, ref(c), a, b, n)


def fork(L, h, c=cache(), a=OK, b=OK, n=3):
    return L.hymt_paged_fork(h, ref(c), a, b, n)


def set_len(L, h, c=cache(), a=OK, b=OK, n=3):
    return L.hymt_paged_set_len(h, ref(c), a, b, n)


def compact(L, h, c=cache()):
    return L.hymt_paged_compact(h, ref(c))


def append(L, h, c=cache(), layer=0, b=batch(), q=OK, q_ld=2048, k=OK, v=OK, kv_ld=512, io=N.F32, heads=16, r=rope(),
           qnw=OK, knw=OK, eps=1e-6, out=OK):
    return L.hymt_rope_append(h, ref(c), layer, ref(b), q, q_ld, k, v, kv_ld, io, heads, ref(r), qnw, knw, eps, out)


def packed(L, h, c=cache(), layer=0, b=batch(), q=OK, heads=16, scale=0.1, out=OK, dt=N.BF16):
    return L.hymt_attn_packed(h, ref(c), layer, ref(b), q, heads, scale, out, dt)


def shared(L, h, c=cache(), layer=0, b=batch(cu=None, rows=3), prefix=128, q=OK, heads=16, scale=0.1, out=OK, dt=N.BF16):
    return L.hymt_attn_shared(h, ref(c), layer, ref(b), prefix, q, heads, scale, out, dt)


CALLS = {f.__name__: f for f in (extend, fork, set_len, compact, append, packed, shared)}
UPKEEP = [extend, fork, set_len]
ROWS = [append, packed, shared]


@pytest.mark.parametrize("name", CALLS)
def test_a_good_call_reaches_the_device_check(ctx, name):
    assert CALLS[name](*ctx) == N.HYMT_E_NO_DEVICE
    assert CALLS[name](ctx[0], None) == N.HYMT_E_ARG
    assert CALLS[name](*ctx, c=None) == N.HYMT_E_ARG


@pytest.mark.parametrize("name", CALLS)
def test_caches(ctx, name):
    f = CALLS[name]
    for bad in [{p: None} for p in ("k", "v", "table", "len", "refs", "work")] + [
            {p: 0} for p in ("layers", "pages", "kv_heads", "seqs", "blocks")] + [
            dict(pages=-1), dict(reserved=1), dict(k=OK + 128), dict(v=OK + 16), dict(table=OK + 2), dict(len=OK + 1),
            dict(refs=OK + 2), dict(work=OK + 2)]:
        assert f(*ctx, c=cache(**bad)) == N.HYMT_E_ARG, bad
    for bad in (dict(dtype=N.F32), dict(dtype=7), dict(head_dim=96), dict(head_dim=256), dict(kv_heads=257),
                dict(seqs=65537), dict(blocks=(1 << 24) + 1), dict(pages=(1 << 28) + 1)):
        assert f(*ctx, c=cache(**bad)) == N.HYMT_E_UNSUPPORTED, bad
    for good in (dict(dtype=N.F16), dict(k=OK + 256), dict(refs=OK + 4), dict(seqs=65536), dict(blocks=1 << 24)):
        assert f(*ctx, c=cache(**good)) == N.HYMT_E_NO_DEVICE, good
    assert f(*ctx, c=cache(head_dim=64), **(dict(r=rope(dim=64)) if f is append else {})) == N.HYMT_E_NO_DEVICE


@pytest.mark.parametrize("f", UPKEEP)
def test_entries(ctx, f):
    assert f(*ctx, a=None) == N.HYMT_E_ARG
    assert f(*ctx, a=OK + 2) == N.HYMT_E_ARG
    assert f(*ctx, b=OK + 2) == N.HYMT_E_ARG
    assert f(*ctx, b=None) == (N.HYMT_E_ARG if f is fork else N.HYMT_E_NO_DEVICE)
    assert f(*ctx, n=-1) == N.HYMT_E_ARG
    assert f(*ctx, n=0) == N.HYMT_E_NO_DEVICE
    assert f(*ctx, n=N.PAGED_BATCH) == N.HYMT_E_NO_DEVICE
    assert f(*ctx, n=N.PAGED_BATCH + 1) == N.HYMT_E_UNSUPPORTED


@pytest.mark.parametrize("f", ROWS)
def test_batches(ctx, f):
    one = dict(cu=None, rows=3)
    own = one if f is shared else {}
    assert f(*ctx, b=None) == N.HYMT_E_ARG
    for bad in (dict(slots=None), dict(slots=OK + 1), dict(cu=OK + 2), dict(n=-1), dict(rows=-1), dict(max_len=-1),
                dict(reserved=1), dict(cu=None, rows=4)):
        assert f(*ctx, b=batch(**{**own, **bad})) == N.HYMT_E_ARG, bad
    assert f(*ctx, b=batch(**{**own, "n": 1025, "rows": 1025})) == N.HYMT_E_UNSUPPORTED
    assert f(*ctx, b=batch(**one)) == N.HYMT_E_NO_DEVICE
    if f is shared:
        assert f(*ctx, b=batch()) == N.HYMT_E_ARG  # packed rows
    else:
        assert f(*ctx, b=batch(rows=(1 << 24) + 1)) == N.HYMT_E_UNSUPPORTED
        assert f(*ctx, b=batch(rows=0)) == N.HYMT_E_NO_DEVICE
        assert f(*ctx, b=batch(rows=1 << 22)) == N.HYMT_E_NO_DEVICE
        assert f(*ctx, b=batch(rows=(1 << 22) + 1)) == N.HYMT_E_UNSUPPORTED
        wide = dict(q_ld=1 << 16) if f is append else {}
        assert f(*ctx, b=batch(rows=1 << 22), heads=64, **wide) == N.HYMT_E_NO_DEVICE  # 2^28 rows of all heads
        assert f(*ctx, b=batch(rows=1 << 22), heads=68, **wide) == N.HYMT_E_UNSUPPORTED


@pytest.mark.parametrize("f", ROWS)
def test_layers_and_heads(ctx, f):
    for bad in (dict(layer=-1), dict(layer=2), dict(heads=0), dict(heads=18), dict(heads=-4)):
        assert f(*ctx, **bad) == N.HYMT_E_ARG, bad
    assert f(*ctx, layer=1) == N.HYMT_E_NO_DEVICE
    wide = dict(q_ld=1 << 16) if f is append else {}
    assert f(*ctx, heads=256, **wide) == N.HYMT_E_NO_DEVICE
    assert f(*ctx, heads=260, **wide) == N.HYMT_E_UNSUPPORTED


def test_append(ctx):
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(r=None), dict(q=OK + 8), dict(k=OK + 8),
                dict(v=OK + 4), dict(out=OK + 8), dict(qnw=OK + 4), dict(knw=OK + 8), dict(q_ld=2040), dict(q_ld=2052),
                dict(kv_ld=504), dict(kv_ld=516), dict(eps=-1.0), dict(eps=float("nan")), dict(r=rope(freq=None)),
                dict(r=rope(freq=OK + 4)), dict(r=rope(interleaved=2)), dict(r=rope(reserved=1)),
                dict(r=rope(scale=float("nan"))), dict(r=rope(scale=float("inf")))):
        assert append(*ctx, **bad) == N.HYMT_E_ARG, bad
    for bad in (dict(io=3), dict(io=-1), dict(r=rope(dim=8)), dict(r=rope(dim=144)), dict(r=rope(dim=-16)),
                dict(c=cache(head_dim=64), r=rope(dim=80))):
        assert append(*ctx, **bad) == N.HYMT_E_UNSUPPORTED, bad
    for good in (dict(qnw=None), dict(knw=None), dict(io=N.F16), dict(io=N.BF16), dict(q_ld=3000), dict(eps=0.0),
                 dict(r=rope(dim=0, freq=None)), dict(r=rope(dim=48, interleaved=1))):
        assert append(*ctx, **good) == N.HYMT_E_NO_DEVICE, good


@pytest.mark.parametrize("f", [packed, shared])
def test_attention(ctx, f):
    for bad in (dict(q=None), dict(out=None), dict(q=OK + 8), dict(out=OK + 8), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert f(*ctx, **bad) == N.HYMT_E_ARG, bad
    assert f(*ctx, dt=N.F32) == N.HYMT_E_UNSUPPORTED
    assert f(*ctx, dt=N.F16) == N.HYMT_E_NO_DEVICE
    assert f(*ctx, scale=-0.5) == N.HYMT_E_NO_DEVICE
    if f is shared:
        for prefix, want in ((-64, N.HYMT_E_ARG), (63, N.HYMT_E_ARG), (100, N.HYMT_E_ARG), (0, N.HYMT_E_NO_DEVICE),
                             (1 << 20, N.HYMT_E_NO_DEVICE)):
            assert shared(*ctx, prefix=prefix) == want, prefix


@pytest.mark.parametrize("dim", [2, 16, 64, 128])
def test_frequencies(dim):
    half = dim // 2
    i = np.arange(half)
    f, s = rope_freqs(dim, 10000.0)
    plain = 10000.0 ** (-2.0 * i / dim)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert s == 1.0
    f, s = rope_freqs(dim, 10000.0, ROPE_LINEAR, 4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-14)
    f, s = rope_freqs(dim, 10000.0, ROPE_NTK, 4.0)
    base = 10000.0 * 4.0 ** (dim / (dim - 2)) if dim > 2 else 10000.0
    np.testing.assert_allclose(f, base ** (-2.0 * i / dim), rtol=1e-13)
    if dim > 2:  # the slowest pair turns 4 times slower
        np.testing.assert_allclose(f[-1], plain[-1] / 4, rtol=1e-13)
    f, s = rope_freqs(dim, 10000.0, ROPE_YARN, 8.0, 4096)
    np.testing.assert_allclose(s, 0.1 * math.log(8.0) + 1, rtol=1e-7)
    turns = 4096 * plain / (2 * math.pi)
    assert ((f <= plain * (1 + 1e-14)) & (f >= plain / 8 * (1 - 1e-14))).all()
    # two pairs of slack: the blend's ends are rounded outwards to whole pairs
    step = 10000.0 ** (4.0 / dim)
    np.testing.assert_allclose(f[turns > 32 * step], plain[turns > 32 * step], rtol=1e-14)
    np.testing.assert_allclose(f[turns < 1 / step], plain[turns < 1 / step] / 8, rtol=1e-14)
    same, s = rope_freqs(dim, 10000.0, ROPE_YARN, 1.0, 4096)
    np.testing.assert_allclose(same, plain, rtol=1e-14)


def test_frequency_refusals():
    f, s = (ctypes.c_double * 8)(), ctypes.c_float()
    call = N.lib().hymt_rope_freqs
    assert call(16, 1e4, ROPE_NONE, 0.0, 0, f, ctypes.byref(s)) == N.HYMT_OK
    for bad in ((0, 1e4, 0, 1.0, 1), (15, 1e4, 0, 1.0, 1), (-2, 1e4, 0, 1.0, 1), (16, 1.0, 0, 1.0, 1),
                (16, math.inf, 0, 1.0, 1), (16, math.nan, 0, 1.0, 1), (16, 1e4, 1, 0.5, 1), (16, 1e4, 2, math.nan, 1),
                (16, 1e4, 3, math.inf, 1), (16, 1e4, 3, 2.0, 0)):
        assert call(*bad, f, ctypes.byref(s)) == N.HYMT_E_ARG, bad
    assert call(16, 1e4, 4, 2.0, 1, f, ctypes.byref(s)) == N.HYMT_E_UNSUPPORTED
    assert call(16, 1e4, -1, 2.0, 1, f, ctypes.byref(s)) == N.HYMT_E_UNSUPPORTED
    assert call(16, 1e4, 0, 1.0, 1, None, ctypes.byref(s)) == N.HYMT_E_ARG
    assert call(16, 1e4, 0, 1.0, 1, f, None) == N.HYMT_E_ARG
