"""Generation with log probabilities where logits have no largest one: a NaN or
+inf among them is no top token, and the generated tokens are those of a
generation without log probabilities all the same."""
import ctypes

import numpy as np
import pytest

import decode

pytestmark = pytest.mark.gpu

TINY = dict(n_layers=1, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000, rope_theta=1e6,
            norm_eps=1e-6, seed=7)


def damage(m, row, scale):
    """The scale of the first block of a row of the vocabulary's matrix, an f16 number's bits."""
    p, n, k = m.matrix(m.n_matrices() - 1)
    assert row < n
    ctypes.memmove(p + row * (k // 32) * 18, np.array([scale], "<u2").tobytes(), 2)


@pytest.mark.parametrize("scale", [0x7E00, 0x7C00, 0xFC00], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("rows", [(0,), (700,), (999, 3, 41)])
@pytest.mark.parametrize("n_top", [0, 5])
def test_tokens_are_those_without_log_probabilities(n_top, rows, scale):
    """A damaged row is a damaged logit; a token of such a row, taken as the next
    input (the matrix holds the embeddings too), leaves NaN alone."""
    with decode.Model(threads=8, **TINY) as m:
        for row in rows:
            damage(m, row, scale)
        m.attach_gpu(0)
        m.set_attention(m.ATTENTION_GPU)
        prompt = np.arange(100, 109, dtype=np.int32)
        for n in (1, 6):
            m.set_logprobs(-1)
            toks, _ = m.generate(prompt, n)
            logits = m.last_logits()
            if n == 1:
                assert not np.isfinite(logits[list(rows)]).any() and np.isfinite(logits).sum() == 1000 - len(rows)
            m.set_logprobs(n_top)
            same, _ = m.generate(prompt, n)
            assert np.array_equal(same, toks)
            assert np.array_equal(m.last_logits(), logits, equal_nan=True)
            lp, ent, top, top_lp = m.last_logprobs(n, n_top)
            if (logits < np.inf).all():
                assert np.isfinite(lp[-1]) and np.isfinite(ent[-1]) and np.all(top[-1, :1] == toks[-1])
            else:  # as mi355x_logprobs has it
                assert np.isnan(lp[-1]) and np.isnan(ent[-1]) and np.all(top[-1] == -1) and np.all(np.isnan(top_lp[-1]))
