"""Model.score's scratch is sized by the rows that are scored, not by the longest
prefill before: scoring two tokens behind a long one takes two rows of logits,
not 256."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a GPU", allow_module_level=True)

from tinyminigo_b200 import synth  # noqa: E402
from tinyminigo_b200.model import Model, ModelConfig  # noqa: E402

VOCAB = 60000


def model():
    cfg = dict(hidden_size=64, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
               head_dim=16, intermediate_size=128, vocab_size=VOCAB, rope_theta=10000.0,
               rms_norm_eps=1e-6, tie_word_embeddings=False)
    mc = ModelConfig(64, 1, 4, 2, 16, 128, 1e-6, 10000.0, VOCAB, [], 0)
    return Model.from_tensors(mc, dict(synth.make_weights(cfg, 7)))


def test_a_short_score_behind_a_long_prefill_takes_little_memory():
    toks = np.random.default_rng(1).integers(0, VOCAB, 600)
    first = model()  # loads every kernel that the calls below use
    first.forward_seq(toks, first.new_cache(700))
    first.score(toks[:2], first.new_cache(16))
    want = first.score(toks, first.new_cache(700))
    m = model()
    c = m.new_cache(700)
    m.forward_seq(toks, c)
    c.reset()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    two = m.score(toks[:2], c)
    torch.cuda.synchronize()
    # 2 rows of 60000 and their scores: half a MB, allocated in 2 MB pieces
    assert free - torch.cuda.mem_get_info()[0] <= 4 << 20
    # and it grows: cut into calls of every size, the scores agree
    assert abs(two.logprobs[0] - want.logprobs[0]) < 1e-3
    at = 2
    while at < 600:
        n = min(at, 600 - at)
        got = m.score(toks[at:at + n], c)
        assert np.abs(got.logprobs - want.logprobs[at:at + n - 1]).max(initial=0) < 1e-3
        assert np.abs(got.entropies - want.entropies[at:at + n]).max() < 1e-3
        at += n
    first.close()
    m.close()
