"""The 4-bit KV cache and scoring through the model: Model.new_cache(bits=4)
in forward_token, forward_seq, decode, generate and generate_batch, and
Model.score on either cache.

What a 4-bit cache changes is which rows the attention sees, so it is tested
against the same attention over those rows: an f32 numpy forward of the model
whose cache rows are quantised (kv4_ref.py) as they are appended.  Rows near a
rounding border may fall on either side of it (the row itself differs in its
last bits between the two forwards), which moves single elements of the cache
by a step, so logits are compared within 5e-2 and the rows by the share that
agrees; paths of the library among themselves within 2e-3 for the same reason
(prefill and decode compute a row in different orders).
"""
import ctypes
import json
from pathlib import Path

import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a GPU", allow_module_level=True)

from tinyminigo_b200 import synth  # noqa: E402
from tinyminigo_b200._lib import TmgError, check, lib  # noqa: E402
from tinyminigo_b200.model import (GenParams, Model, ModelConfig, generate,  # noqa: E402
                                   generate_batch)


def cfg_obj(cfg):
    return ModelConfig(cfg["hidden_size"], cfg["num_hidden_layers"], cfg["num_attention_heads"],
                       cfg["num_key_value_heads"], cfg["head_dim"], cfg["intermediate_size"],
                       cfg["rms_norm_eps"], cfg["rope_theta"], cfg["vocab_size"], [], 0)


def small(d, heads=4, kv=2, layers=2, vocab=500):
    return dict(hidden_size=heads * d, num_hidden_layers=layers, num_attention_heads=heads,
                num_key_value_heads=kv, head_dim=d, intermediate_size=256, vocab_size=vocab,
                rope_theta=10000.0, rms_norm_eps=1e-6, tie_word_embeddings=False)


def widen(b):
    return (np.asarray(b).astype(np.uint32) << 16).view(np.float32)


class NumpyModel:
    """A Llama-style forward in f32 whose cache rows are what 4 bits stand for."""

    def __init__(self, cfg, w, quantise=True):
        self.cfg, self.quantise = cfg, quantise
        self.w = {k: widen(v) if v.dtype == np.uint16 else np.asarray(v, np.float32)
                  for k, v in w.items()}
        self.k = [[] for _ in range(cfg["num_hidden_layers"])]
        self.v = [[] for _ in range(cfg["num_hidden_layers"])]

    def norm(self, x, w):
        return x / np.sqrt(np.mean(x * x) + self.cfg["rms_norm_eps"]) * w

    def step(self, token):
        c, w = self.cfg, self.w
        d, nq, nkv = c["head_dim"], c["num_attention_heads"], c["num_key_value_heads"]
        pos = len(self.k[0])
        inv = 1.0 / c["rope_theta"] ** (np.arange(0, d, 2) / d)
        cs, sn = np.cos(pos * inv), np.sin(pos * inv)

        def rope(x):
            a, b = x[..., :d // 2], x[..., d // 2:]
            return np.concatenate([a * cs - b * sn, a * sn + b * cs], -1).astype(np.float32)

        def stored(x):
            return R.values(*R.quantise(x)).astype(np.float32) if self.quantise else x

        x = w["model.embed_tokens.weight"][token]
        for i in range(c["num_hidden_layers"]):
            p = f"model.layers.{i}."
            h = self.norm(x, w[p + "input_layernorm.weight"])
            q = rope((w[p + "self_attn.q_proj.weight"] @ h).reshape(nq, d))
            k = rope((w[p + "self_attn.k_proj.weight"] @ h).reshape(nkv, d))
            v = (w[p + "self_attn.v_proj.weight"] @ h).reshape(nkv, d)
            self.k[i].append(stored(k))
            self.v[i].append(stored(v))
            o, _ = R.attention(q, np.stack(self.k[i]), np.stack(self.v[i]))
            x = x + w[p + "self_attn.o_proj.weight"] @ o.reshape(-1).astype(np.float32)
            h = self.norm(x, w[p + "post_attention_layernorm.weight"])
            g = w[p + "mlp.gate_proj.weight"] @ h
            x = x + w[p + "mlp.down_proj.weight"] @ (g / (1 + np.exp(-g)) *
                                                     (w[p + "mlp.up_proj.weight"] @ h))
        h = self.norm(x, w["model.norm.weight"])
        return w.get("lm_head.weight", w["model.embed_tokens.weight"]) @ h


@pytest.mark.parametrize("d,heads,kv", [(16, 4, 2), (32, 4, 4), (64, 8, 2), (128, 4, 1)])
def test_forward_token_sees_quantised_rows(d, heads, kv):
    cfg = small(d, heads, kv)
    w = dict(synth.make_weights(cfg, 11 + d))
    m = Model.from_tensors(cfg_obj(cfg), w)
    ref = NumpyModel(cfg, w)
    c = m.new_cache(37, bits=4)
    toks = np.random.default_rng(d).integers(0, cfg["vocab_size"], 30)
    for t in toks:
        a, b = m.forward_token(int(t), c), ref.step(int(t))
        assert np.abs(a - b).max() < 5e-2
    assert c.len() == 30
    same = total = 0
    for i in range(cfg["num_hidden_layers"]):
        for got, want in ((c.keys_flat(i), ref.k[i]), (c.values_flat(i), ref.v[i])):
            want = np.stack(want).reshape(30, -1)
            same += int(np.sum(np.abs(got - want) <= 1e-6 * np.abs(want).max()))
            total += want.size
    assert same >= 0.98 * total
    m.close()


def test_rows_are_the_operators_rows():
    # the rows that a step writes are bit for bit what tmg_op_kv4_append makes
    # of the f32 cache's rows: one layer, so both caches hold the same keys
    cfg = small(64, 8, 2, layers=1)
    w = dict(synth.make_weights(cfg, 5))
    m = Model.from_tensors(cfg_obj(cfg), w)
    for prompt in (0, 12, 20):
        toks = np.random.default_rng(prompt).integers(0, cfg["vocab_size"], 20)
        a, b = m.new_cache(64), m.new_cache(64, bits=4)
        for c in (a, b):
            if prompt:
                m.forward_seq(toks[:prompt], c)
            for t in toks[prompt:]:
                m.forward_token(int(t), c)
        for get in ("keys_flat", "values_flat"):
            x = getattr(a, get)(0).reshape(20, 2, 64)
            want = R.values(*R.quantise(x)).astype(np.float32).reshape(20, -1)
            assert np.array_equal(getattr(b, get)(0), want)
        a.close()
        b.close()
    m.close()


def test_prefill_in_pieces_and_steps_agree():
    cfg = small(64, 8, 2)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 3)))
    toks = np.random.default_rng(2).integers(0, cfg["vocab_size"], 200).tolist()
    whole, cut, step = (m.new_cache(256, bits=4) for _ in range(3))
    a = m.forward_seq(toks, whole)
    m.forward_seq(toks[:70], cut)
    m.forward_seq(toks[70:71], cut)
    b = m.forward_seq(toks[71:], cut)
    for t in toks:
        s = m.forward_token(t, step)
    assert np.abs(a - b).max() < 2e-3 and np.abs(a - s).max() < 2e-3
    # truncate and append again: the same tokens give the same state
    whole.truncate(150)
    assert whole.len() == 150
    assert np.abs(m.forward_seq(toks[150:], whole) - a).max() < 2e-3
    whole.reset()
    assert whole.len() == 0 and whole.keys_flat(0).shape == (0, 128)
    m.close()


def test_generate_decode_and_batch_agree():
    cfg = small(32, 4, 2)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 9)))
    rng = np.random.default_rng(4)
    prompts = rng.integers(0, cfg["vocab_size"], (3, 11))
    one = [generate(m, p, GenParams(max_tokens=24), cache=m.new_cache(64, bits=4)).tokens
           for p in prompts]
    batch = generate_batch(m, prompts, [GenParams(max_tokens=24)] * 3,
                           cache=m.new_cache(64, n_streams=3, bits=4))
    agree = np.mean([x == y for a, b in zip(one, batch) for x, y in zip(a, b)])
    assert agree >= 0.9  # near-ties of a random model aside
    c = m.new_cache(64, bits=4)
    m.forward_seq(prompts[0], c)
    ids = m.decode(one[0][0], c, 23)
    assert ids.shape == (1, 23) and c.len() == 11 + 23
    assert np.mean(ids[0] == np.asarray(one[0][1:])) >= 0.9
    # sampling takes the cache too
    s = GenParams(max_tokens=10, temperature=0.7, top_k=20, top_p=0.9)
    out = generate(m, prompts[0], s, cache=m.new_cache(64, bits=4))
    assert len(out.tokens) == 10
    # full to the last position
    c = m.new_cache(21, bits=4)
    assert len(generate(m, prompts[0], GenParams(max_tokens=10), cache=c).tokens) == 10
    with pytest.raises(TmgError) as e:
        generate(m, prompts[0], GenParams(max_tokens=11), cache=c)
    assert e.value.code == -4
    m.close()


def test_refusals_of_a_4_bit_cache():
    cfg = small(64, 8, 2)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 1)))
    with pytest.raises(ValueError):
        m.new_cache(16, bits=8)
    h = ctypes.c_void_p()
    assert lib().tmg_kv_create_q4(m._h, 0, 16, ctypes.byref(h)) == -1
    assert lib().tmg_kv_create_q4(m._h, 1, 0, ctypes.byref(h)) == -1
    assert lib().tmg_kv_create_q4(m._h, 1, 2**31, ctypes.byref(h)) == -1
    c = m.new_cache(16, bits=4)
    with pytest.raises(TmgError):
        m.trace_decode([1], c)
    with pytest.raises(TmgError):
        m.score([1, 2], c, top=65)
    with pytest.raises(TmgError):
        m.score([1, 500], c)
    with pytest.raises(TmgError) as e:
        m.score([1] * 17, c)
    assert e.value.code == -4 and c.len() == 0
    m.close()
    # a head dim and a group that the 4-bit kernels do not take
    for odd in (small(48, 4, 2), small(16, 34, 2)):
        x = Model.from_tensors(cfg_obj(odd), dict(synth.make_weights(odd, 1)))
        with pytest.raises(TmgError):
            x.new_cache(16, bits=4)
        x.close()


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("T", [1, 2, 70, 300])
def test_score(bits, T):
    # against the last-row distributions of forward_seq over the same tokens'
    # prefixes (the same kernels up to the LM head, so the same cache rows; a
    # row from another kernel may fall on the other side of a rounding border
    # and move an element by a whole step)
    cfg = small(64, 8, 2, vocab=1003)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 21)))
    toks = np.random.default_rng(T).integers(0, 1003, T)
    c, s = m.new_cache(310, bits=bits), m.new_cache(310, bits=bits)
    got = m.score(toks, c, top=5)
    assert c.len() == T
    assert got.logprobs.shape == (T - 1,) and got.top_ids.shape == (T, 5)
    tol = 1e-3
    for t in range(T):
        s.reset()
        x = m.forward_seq(toks[:t + 1], s).astype(np.float64)
        lp = x - x.max()
        lp -= np.log(np.exp(lp).sum())
        assert abs(got.entropies[t] + (np.exp(lp) * lp).sum()) < tol
        assert np.all(np.abs(got.top_logprobs[t] - np.sort(lp)[::-1][:5]) < tol)
        assert np.all(np.abs(lp[got.top_ids[t]] - got.top_logprobs[t]) < tol)
        if t + 1 < T:
            assert abs(got.logprobs[t] - lp[toks[t + 1]]) < tol
    # scoring goes on where it stopped
    if T > 2:
        c.truncate(T - 2)
        again = m.score(toks[T - 2:], c)
        assert abs(again.logprobs[0] - got.logprobs[T - 2]) < tol
    m.close()


def test_score_beyond_a_chunk():
    # 4096 positions go through the layers at a time, 256 rows of logits; cut
    # elsewhere, the scores agree
    cfg = small(64, 4, 2, vocab=307)
    m = Model.from_tensors(cfg_obj(cfg), dict(synth.make_weights(cfg, 4)))
    toks = np.random.default_rng(8).integers(0, 307, 4500)
    a = m.score(toks, m.new_cache(4500), top=3)
    c = m.new_cache(4500)
    b1, b2 = m.score(toks[:4001], c, top=3), m.score(toks[4001:], c, top=3)
    assert c.len() == 4500
    assert np.abs(a.logprobs[:4000] - b1.logprobs).max() < 1e-3
    assert np.abs(a.logprobs[4001:] - b2.logprobs).max() < 1e-3
    assert np.abs(a.entropies - np.concatenate([b1.entropies, b2.entropies])).max() < 1e-3
    assert np.abs(a.top_logprobs - np.concatenate([b1.top_logprobs, b2.top_logprobs])).max() < 1e-3
    m.close()


def test_perplexity_of_a_4_bit_cache_is_near():
    # the use that the operators have together: a text scored with its cache in
    # 32 bits and in 4
    d = json.loads((Path(__file__).resolve().parent / "golden" / "hf_c1.json").read_text())
    cfg = synth.CONFIGS["c1"]
    m = Model.from_tensors(cfg_obj(cfg), synth.make_weights(cfg, d["weight_seed"]))
    toks = np.random.default_rng(0).integers(0, cfg["vocab_size"], 500)
    full, four = (m.score(toks, m.new_cache(512, bits=b)) for b in (32, 4))
    assert np.isfinite(full.logprobs).all() and np.isfinite(four.logprobs).all()
    assert abs(np.log(four.perplexity()) - np.log(full.perplexity())) < 0.02
    with pytest.raises(TmgError):
        check(lib().tmg_score(None, None, 0, None, 1, 0, None, None, None, None))
    m.close()
