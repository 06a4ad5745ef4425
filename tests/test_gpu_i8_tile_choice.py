"""HYMT_HIP_I8_TILE through hymt_model_prefill: an unknown name is refused before
anything is enqueued, a tile's name gives the bits of the planned tiles."""
import numpy as np
import pytest

from hymt2sharp_amd import HipBackend
from hymt2sharp_amd import _native as N
from hymt2sharp_amd import synth as S
from hymt2sharp_amd.model import ModelConfig

pytestmark = pytest.mark.gpu


def test_a_prompt_under_a_forced_tile(hip_available, monkeypatch):
    monkeypatch.delenv("HYMT_HIP_I8_TILE", raising=False)
    cfg = ModelConfig(num_layers=1, vocab_size=64)
    t = S.random_model(1, cfg, {"attn": N.W_Q4_K, "ffn": N.W_Q4_K, "embd": N.W_Q6_K, "out": N.W_Q6_K})
    be = HipBackend(0)
    try:
        be.LoadModel(t, cfg, max_tokens=128, int8=True)
        m, toks = be._model, list(range(40))

        def logits():
            be.SetCacheLen(0)
            m.prefill(toks, 0)
            be.sync()
            return be.download(np.empty(cfg.vocab_size, np.float32), m.logits)

        want = logits()
        be.upload(m.logits, np.zeros(cfg.vocab_size, np.float32))
        be.SetCacheLen(0)
        monkeypatch.setenv("HYMT_HIP_I8_TILE", "64x65")
        ids = np.asarray(toks, np.int32)
        assert be._lib.hymt_model_prefill(m._native, ids.ctypes.data, len(toks), 0, m.logits,
                                          N.PREFILL_INT8) == N.HYMT_E_ARG
        be.sync()
        assert not be.download(np.empty(cfg.vocab_size, np.float32), m.logits).any()
        for tile in ("16x16", "64x64", "128x128"):
            monkeypatch.setenv("HYMT_HIP_I8_TILE", tile)
            np.testing.assert_array_equal(logits(), want)
    finally:
        be.Dispose()
