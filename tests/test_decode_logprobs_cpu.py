"""What the decode harness refuses of its log probabilities."""
import pytest

import decode

TINY = dict(n_layers=1, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, ffn=64, vocab=50, rope_theta=1e4,
            norm_eps=1e-5, seed=1)


def test_top_tokens_are_checked():
    with decode.Model(threads=1, **TINY) as m:
        for n in (-1, 0, 50):
            m.set_logprobs(n)
        for n in (-2, 51, 65):
            with pytest.raises(RuntimeError, match="n_top"):
                m.set_logprobs(n)
    with decode.Model(threads=1, **dict(TINY, vocab=100)) as m:
        m.set_logprobs(64)
        with pytest.raises(RuntimeError, match="n_top"):
            m.set_logprobs(65)


def test_they_need_attention_on_the_gpu():
    calls = []

    def gemv(*args):
        calls.append(args)

    with decode.Model(threads=1, **TINY) as m:
        m.set_logprobs(0)
        with pytest.raises(RuntimeError, match="attention on the GPU"):
            m.generate(decode.prompt_tokens(3, 50, 1), 1, cpu_gemv=gemv)
        assert not calls


def test_none_before_a_generation():
    with decode.Model(threads=1, **TINY) as m:
        for n in (0, 1):
            with pytest.raises(RuntimeError, match="no such"):
                m.last_logprobs(n)
