"""Log probabilities of the decode harness's generated tokens, against the
logits that it keeps of the last one.

With u = 2^-24 and d = max - x: exp2's argument is off by 3 u d log2 e, the power
by 1 u, a sum of V terms by less than (V / 256 + 64) u of itself (its chain in a
thread and the joins); so log p is off by (3 mean d + 4 + V / 256 + 64) u, d itself and the last
rounding by 3 u |log p|, and the entropy by twice that and the entropy's own roundings."""
import numpy as np
import pytest

import decode
import layer_ref

pytestmark = pytest.mark.gpu

TINY = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000, rope_theta=1e6,
            norm_eps=1e-6, seed=7)
U = 2.0 ** -24


@pytest.mark.parametrize("n_top", [0, 1, 5, 64])
@pytest.mark.parametrize("vocab", [65, 1000, 20000])
def test_generated_tokens(n_top, vocab):
    cfg = dict(TINY, vocab=vocab)
    with decode.Model(threads=8, **cfg) as m:
        m.attach_gpu(0)
        m.set_attention(m.ATTENTION_GPU)
        p = decode.prompt_tokens(20, vocab, 2)
        toks, _ = m.generate(p, 12)
        logits = m.last_logits()
        m.set_logprobs(n_top)
        same, _ = m.generate(p, 12)
        assert np.array_equal(same, toks) and np.array_equal(m.last_logits(), logits)
        lp, ent, top, top_lp = m.last_logprobs(12, n_top)
        with pytest.raises(RuntimeError, match="no such"):
            m.last_logprobs(12, max(n_top, 1) + 1)
        with pytest.raises(RuntimeError, match="no such"):
            m.last_logprobs(11)
        # the last token's are those of the logits
        x = logits[None].astype(np.float64)
        ref, ref_ent = layer_ref.logprobs(x, 1.0)
        mean = float((np.exp(ref) * (x.max() - x)).sum())
        sums = (3 * mean + 4 + vocab / 256 + 64) * U
        order = np.lexsort((np.arange(vocab), -x[0]))[:n_top]
        assert np.array_equal(top[-1], order)
        assert np.all(np.abs(top_lp[-1] - ref[0, order]) <= sums + 3 * U * np.abs(ref[0, order]))
        assert abs(lp[-1] - ref[0, toks[-1]]) <= sums + 3 * U * abs(ref[0, toks[-1]])
        assert abs(ent[-1] - ref_ent[0]) <= 2 * sums * (1 + mean) + 3 * U * abs(ref_ent[0])
        m.generate(p, 1)
        one = m.last_logprobs(1, n_top)
        assert one[0][0] == lp[0] and one[1][0] == ent[0]
        assert np.array_equal(one[2][0], top[0]) and np.array_equal(one[3][0], top_lp[0])
        if n_top:
            assert np.array_equal(top[:, 0], toks) and np.array_equal(top_lp[:, 0], lp)
        m.set_logprobs(-1)
        back, _ = m.generate(p, 12)
        assert np.array_equal(back, toks) and np.array_equal(m.last_logits(), logits)
        with pytest.raises(RuntimeError, match="no such"):
            m.last_logprobs(12)
