"""The 8-bit integer operators in the order a prompt's layer runs them: the chain
against plain references stage by stage, recorded and replayed, on two contexts at
once, and as hymt_model_prefill with HYMT_PREFILL_INT8.

Each stage of the chain is checked from what the stage before it left on the
GPU, with the bounds of the operators' own tests.

The model's logits against the fp32 oracle.  A row coded in 8 bits is off by a
uniform error of +- scale / 2, relative to the row's root mean square
(a / rms) / (127 sqrt(12)) = crest / 440, and a product of two such rows by the two in
quadrature.  Crests: 4 for normal rows of 2048 (0.9 %), up to 20 for the rows of
silu(g) u (4.5 %), 2-4 for weights (0.9 %).  A layer's attention branch (q/k/v, then o)
is then off by up to 1.8 %, its FFN branch by 1.3 % through gate and up, doubled at
most by silu's slope and the product, and 4.6 % through down: 5.3 %; two layers,
added in quadrature to the residual they share: 8 %.  Bound on the 2-norm: 10 %."""
import numpy as np
import pytest

from hymt2sharp_amd import BF16, F16, F32, HipBackend
from hymt2sharp_amd import _native as N
from hymt2sharp_amd import synth as S
from hymt2sharp_amd.model import DeviceModel, ModelConfig, Tensor
from oracle.model import OracleModel
from tests.i8_cases import U16, U32, Room, bf16_bits, bf16_val, codes, codes_of, norm_rows, product, scales

pytestmark = pytest.mark.gpu

CFG = ModelConfig(num_layers=2, vocab_size=512)


@pytest.fixture
def be(hip_available):
    b = HipBackend(0)
    yield b
    b.Dispose()


class Chain:
    """x += d0; norm; q/k/v; (ao); codes; o -> d1; x2 = x + d1; norm; gate/up;
    codes; down onto x2."""

    H, F, K = 512, 768, 640  # hidden, ffn, attention width

    def __init__(self, be, seed, m):
        self.be, self.m, self.r = be, m, Room(be)
        H, F, K, r = self.H, self.F, self.K, self.r
        rng = np.random.default_rng(seed)
        std = lambda n, k, s: (codes(seed + s, n, k), scales(seed + s, n, 2e-4, 5e-4))
        self.w = {"qkv": std(K + 130, H, 1), "o": std(H, K, 2), "gate": std(F, H, 3), "up": std(F, H, 4),
                  "down": std(H, F, 5)}
        self.dw = {n: (r.put(q), r.put(s)) for n, (q, s) in self.w.items()}
        self.x0 = rng.standard_normal((m, H)).astype(np.float32)
        self.d0 = bf16_bits(rng.standard_normal((m, H)))
        self.ao = bf16_bits(rng.standard_normal((m, K)))
        self.g = [rng.uniform(0.8, 1.2, H).astype(np.float32) for _ in range(2)]
        self.a0, self.aao, self.ag = r.put(self.d0), r.put(self.ao), [r.put(g) for g in self.g]
        self.ax0 = r.put(self.x0)
        z = lambda n, dt: r.put(np.zeros((m, n), dt))
        self.x, self.x2 = z(H, np.float32), z(H, np.float32)
        self.q = [z(H, np.int8), z(K, np.int8), z(H, np.int8), z(F, np.int8)]
        self.s = [z(1, np.float32) for _ in range(4)]
        self.qkv, self.d1, self.act, self.y = z(K + 130, np.uint16), z(H, np.uint16), z(F, np.uint16), z(H, np.float32)
        self.one, self.tmp = r.put(np.ones(H, np.float32)), z(H, np.int8)

    def run(self):
        be, m, H, F, K, w, q, s = self.be, self.m, self.H, self.F, self.K, self.dw, self.q, self.s
        gemm = lambda n, rows, k, i, y, **kw: be.gemm_i8(*w[n], rows, k, q[i], s[i], m, y, **kw)
        be.rows_rmsnorm_i8(self.x, m, H, self.ag[0], 1e-5, q[0], s[0], add=self.a0)
        gemm("qkv", K + 130, H, 0, self.qkv, out_bf16=True)
        be.to_i8(self.aao, m, K, q[1], s[1], x_dtype=N.BF16)
        gemm("o", H, K, 1, self.d1, out_bf16=True)
        be.rows_rmsnorm_i8(self.x, m, H, self.ag[1], 1e-5, q[2], s[2], add=self.d1)
        be.gemm_i8_swiglu(*w["gate"], *w["up"], F, H, q[2], s[2], m, self.act)
        be.to_i8(self.act, m, F, q[3], s[3], x_dtype=N.BF16)
        gemm("down", H, F, 3, self.x, accumulate=True)

    def reset(self):
        """The residual as the step before leaves it, on the context's stream."""
        N.check(self.be._lib.hymt_memcpy(self.be.handle, self.x, self.ax0, self.x0.nbytes, 2))

    def got(self):
        m, g = self.m, self.r.get
        widths = (self.H, self.K, self.H, self.F)
        return {"q": [g(p, np.empty((m, n), np.int8)) for p, n in zip(self.q, widths)],
                "s": [g(p, np.empty(m, np.float32)) for p in self.s],
                "qkv": g(self.qkv, np.empty((m, self.K + 130), np.uint16)),
                "d1": g(self.d1, np.empty((m, self.H), np.uint16)),
                "act": g(self.act, np.empty((m, self.F), np.uint16)), "x": g(self.x, self.x0)}

    def check(self, o):
        def row_codes(i, v):
            q, a = codes_of(v)
            np.testing.assert_array_equal(o["q"][i], q)
            np.testing.assert_array_equal(o["s"][i], (a / 127.0).astype(np.float32))

        def norm(i, x, add):
            h, q, s = norm_rows(x, add, self.g[i // 2], 1e-5)
            np.testing.assert_array_equal(o["q"][i], q)
            assert (np.abs(o["s"][i] - s) <= U32 * (1 + 2.0 ** -10) * s).all()
            return h

        def bf16_product(name, got, i):
            y = product(*self.w[name], o["q"][i], o["s"][i])
            assert (np.abs(bf16_val(got) - y) <= np.abs(y) * U16 * (1 + 2.0 ** -10)).all()

        h = norm(0, self.x0, bf16_val(self.d0))
        bf16_product("qkv", o["qkv"], 0)
        row_codes(1, bf16_val(self.ao))
        bf16_product("o", o["d1"], 1)
        h = norm(2, h, bf16_val(o["d1"]))
        g, u = (product(*self.w[n], o["q"][2], o["s"][2]) for n in ("gate", "up"))
        y = g / (1 + np.exp(-g)) * u
        tol = np.abs(y) * (U16 + (5 * np.abs(g) + 16) * U32) * (1 + 2.0 ** -7) + 2.0 ** -125
        assert (np.abs(bf16_val(o["act"]) - y) <= tol).all()
        row_codes(3, bf16_val(o["act"]))
        v = product(*self.w["down"], o["q"][3], o["s"][3])
        y = h.astype(np.float64) + v
        assert (np.abs(o["x"] - y) <= 2.01 * U32 * np.abs(v) + U32 * np.abs(y)).all()


def same(a, b):
    for k in a:
        for p, q in zip(a[k], b[k]):
            np.testing.assert_array_equal(p, q)


@pytest.mark.parametrize("m", [1, 5, 33, 130])
def test_a_layers_chain(be, m):
    c = Chain(be, m, m)
    c.reset()
    c.run()
    c.check(c.got())
    c.r.close()


def test_recorded_chain_replays_exactly(be):
    """Replays with eager work of other shapes and synchronisations between
    them; two recordings on one context."""
    a, b = Chain(be, 1, 40), Chain(be, 2, 3)
    want = []
    for c in (a, b):
        c.reset()
        c.run()
        want.append(c.got())
        c.check(want[-1])
    graphs = []
    for c in (a, b):
        be.graph_begin()
        c.run()
        graphs.append(be.graph_end())
    for rep in range(4):
        for c, g, w in ((a, graphs[0], want[0]), (b, graphs[1], want[1])):
            c.reset()
            be.graph_launch(g)
            if rep % 2:
                be.rows_rmsnorm_i8(c.one, 1, c.H, c.one, 1e-5, c.tmp, c.y)  # other eager work
                c.reset()
                be.graph_launch(g)
            same(c.got(), w)
    for g in graphs:
        be.graph_destroy(g)
    a.r.close()
    b.r.close()


def test_two_contexts_at_once(be):
    """The calls use no workspace: two contexts' streams run side by side."""
    other = HipBackend(0)
    try:
        cs = [Chain(be, 3, 70), Chain(other, 3, 70)]
        for c in cs:
            c.reset()
            c.be.sync()
        for c in cs:  # enqueued on both streams before either is waited for
            c.run()
        got = [c.got() for c in cs]
        cs[0].check(got[0])
        same(*got)
        for c in cs:
            c.r.close()
    finally:
        other.Dispose()


def test_kernels_are_timed_by_name(be):
    c = Chain(be, 4, 9)
    be.timing_enable(2)
    c.reset()
    c.run()
    be.sync()
    counts = {k: be.timing(k)[0] for k in ("gemm_i8_out_f32", "gemm_i8_out_bf16", "gemm_i8_swiglu", "to_i8",
                                           "rows_rmsnorm_i8")}
    assert counts == {"gemm_i8_out_f32": 1, "gemm_i8_out_bf16": 2, "gemm_i8_swiglu": 1, "to_i8": 2, "rows_rmsnorm_i8": 2}
    be.timing_enable(0)
    c.r.close()


# ---- the model -----------------------------------------------------------------------


def mixed_model(seed):
    """Layer 1 has q, k, v and gate, up as separate matrices (their types differ)."""
    t = S.random_model(seed, CFG, {"attn": [N.W_Q4_K, N.W_Q8_0], "ffn": [N.W_Q6_K, N.W_Q4_K], "embd": N.W_Q6_K,
                                   "out": N.W_Q6_K})
    for name, wt in (("blk.1.attn_v.weight", N.W_F16), ("blk.1.ffn_up.weight", N.W_Q8_0)):
        t[name] = Tensor(wt, t[name].rows, t[name].cols, S.random_weight(77, wt, t[name].rows, t[name].cols))
    return t


def logits(be):
    return be.download(np.empty(CFG.vocab_size, np.float32), be._model.logits)


@pytest.mark.parametrize("n", [2, 70, 2100])
def test_native_int8_prefill_equals_composed_calls(be, n):
    """One hymt_model_prefill call (2048-row chunks) against the same calls
    one by one: the same logits and cache rows, bit for bit."""
    be.LoadModel(mixed_model(8), CFG, max_tokens=n + 64, kv_dtype=BF16, int8=True)
    m = be._model
    toks = [int(x) for x in np.random.default_rng(n).integers(0, CFG.vocab_size, n)]
    m.prefill(toks, 0)
    be.sync()
    native, kv = logits(be), [be.ReadKv(l, 0, n) for l in range(CFG.num_layers)]
    assert np.isfinite(native).all() and native.any()
    be.upload(m.logits, np.zeros(CFG.vocab_size, np.float32))
    for i in range(0, n, DeviceModel.PREFILL_CHUNK):
        m.prefill_composed_i8(toks[i:i + DeviceModel.PREFILL_CHUNK], i)
    be.sync()
    np.testing.assert_array_equal(native, logits(be))
    for l in range(CFG.num_layers):
        for a, b in zip(be.ReadKv(l, 0, n), kv[l]):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("kv,m", [(BF16, 40), (F16, 70)])
def test_int8_forward_against_the_oracle(be, kv, m):
    t = mixed_model(4)
    om = OracleModel(CFG, t, 128, kv)
    be.LoadModel(t, CFG, max_tokens=128, kv_dtype=kv, int8=True)
    toks = [int(x) for x in np.random.default_rng(m).integers(0, CFG.vocab_size, m)]
    for got, ref in ((be.ForwardStep(toks, 0), om.forward(toks, 0)), (be.ForwardStep([11], m), om.step(11, m)),
                     (be.ForwardStep([3, 4, 5], m + 1), [om.step(x, m + 1 + i) for i, x in enumerate((3, 4, 5))][-1])):
        err = np.linalg.norm(got - ref) / np.linalg.norm(ref)
        print(f"int8 prefill m={m} rel {err:.2e}", flush=True)
        assert err <= 0.1


def test_int8_prefill_refusals(be):
    cfg = ModelConfig(num_layers=1, vocab_size=64)
    t = S.random_model(1, cfg, {"attn": N.W_Q4_K, "ffn": N.W_Q4_K, "embd": N.W_Q6_K, "out": N.W_Q6_K})
    be.LoadModel(t, cfg, max_tokens=128)  # bf16 copies, no codes
    m = be._model
    call = lambda flags, n=2: be._lib.hymt_model_prefill(m._native, np.zeros(n, np.int32).ctypes.data, n, 0, m.logits,
                                                         flags)
    assert call(N.PREFILL_INT8) == N.HYMT_E_STATE
    assert call(N.PREFILL_INT8, 1) == N.HYMT_E_STATE
    assert call(N.PREFILL_INT8 | N.PREFILL_GATE_UP_F32) == N.HYMT_E_ARG
    assert call(4) == N.HYMT_E_ARG
    assert call(0) == N.HYMT_OK
    for w in be._model._weights:
        be.weight_i8(w)
    assert call(N.PREFILL_INT8) == N.HYMT_OK  # codes beside the bf16 copies: either runs
    be.graph_begin()
    assert call(N.PREFILL_INT8) == N.HYMT_E_STATE
    with pytest.raises(N.InvalidOperationError):
        be.graph_end()
    be.graph_begin()
    with pytest.raises(N.InvalidOperationError):
        be.weight_i8(be._model._weights[0])
    with pytest.raises(N.InvalidOperationError):
        be.graph_end()


def test_int8_model_over_an_fp32_cache_runs_decode_steps(be):
    cfg = ModelConfig(num_layers=1, vocab_size=64)
    t = S.random_model(2, cfg, {"attn": N.W_Q4_K, "ffn": N.W_Q4_K, "embd": N.W_Q6_K, "out": N.W_Q6_K})
    be.LoadModel(t, cfg, max_tokens=64, kv_dtype=F32, int8=True)
    a = be.ForwardStep([1, 2, 3], 0)
    be.SetCacheLen(0)
    b = [be.ForwardStep([x], i) for i, x in enumerate((1, 2, 3))][-1]
    np.testing.assert_array_equal(a, b)
