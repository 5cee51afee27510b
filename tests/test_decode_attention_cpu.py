"""What the decode harness refuses of its attention modes."""
import pytest

import decode

TINY = dict(n_layers=1, hidden=64, n_heads=2, n_kv_heads=1, head_dim=32, ffn=64, vocab=100, rope_theta=1e4,
            norm_eps=1e-5, seed=1)


def test_attention_mode_is_checked():
    with decode.Model(threads=1, **TINY) as m:
        m.set_attention(m.ATTENTION_HOST)
        with pytest.raises(RuntimeError, match="head_dim"):
            m.set_attention(m.ATTENTION_GPU)
        with pytest.raises(RuntimeError, match="unknown mode"):
            m.set_attention(7)
    with decode.Model(threads=1, **dict(TINY, head_dim=64)) as m:
        m.set_attention(m.ATTENTION_GPU)
        with pytest.raises(RuntimeError, match="attach_gpu"):
            m.generate(decode.prompt_tokens(3, 100, 1), 1)
