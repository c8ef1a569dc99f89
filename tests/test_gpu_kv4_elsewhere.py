"""The 4-bit cache and scoring where other modes of the library meet them: the
fused group (refused, by name) and int8 weights (TMG_I8=1)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a GPU", allow_module_level=True)

from test_gpu_kv4_model import cfg_obj, small  # noqa: E402

from tinyminigo_b200 import synth  # noqa: E402
from tinyminigo_b200._lib import lib  # noqa: E402
from tinyminigo_b200.model import Model  # noqa: E402


def test_a_fused_group_refuses_a_4_bit_cache_by_name():
    cfg = small(64, 8, 2)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 1)))
    c = m.new_cache(16, bits=4)
    uid = (ctypes.c_uint8 * 128)()
    assert lib().tmg_fused_group_init(m._h, c._h, uid, 0, 2) == -1
    assert "4-bit" in m.last_error()
    assert np.isfinite(m.forward_token(3, c)).all() and c.len() == 1
    m.close()


@pytest.mark.parametrize("bits", [32, 4])
def test_score_with_int8_weights(bits, monkeypatch):
    # as test_score: the last-row distributions of forward_seq over the prefixes,
    # by the same kernels up to the LM head
    monkeypatch.setenv("TMG_I8", "1")
    cfg = small(64, 8, 2, vocab=1003)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 21)))
    toks = np.random.default_rng(5).integers(0, 1003, 40)
    c, s = m.new_cache(64, bits=bits), m.new_cache(64, bits=bits)
    got = m.score(toks, c, top=5)
    for t in range(40):
        s.reset()
        x = m.forward_seq(toks[:t + 1], s).astype(np.float64)
        lp = x - x.max()
        lp -= np.log(np.exp(lp).sum())
        assert abs(got.entropies[t] + (np.exp(lp) * lp).sum()) < 1e-3
        assert np.all(np.abs(got.top_logprobs[t] - np.sort(lp)[::-1][:5]) < 1e-3)
        if t + 1 < 40:
            assert abs(got.logprobs[t] - lp[toks[t + 1]]) < 1e-3
    m.close()


def test_steps_with_int8_weights_over_a_4_bit_cache(monkeypatch):
    # 0.25: the int8 path's own noise, as in test_gpu_i8.py
    monkeypatch.setenv("TMG_I8", "1")
    cfg = small(64, 8, 2)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 3)))
    toks = np.random.default_rng(6).integers(0, cfg["vocab_size"], 30)
    a, b = m.new_cache(64), m.new_cache(64, bits=4)
    for t in toks:
        x, y = m.forward_token(int(t), a), m.forward_token(int(t), b)
        assert np.isfinite(y).all() and np.abs(x - y).max() < 0.25
    m.close()
