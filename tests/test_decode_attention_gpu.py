"""The decode harness with attention on the GPU: plan, rotation and store, and
attention over f16 pages in every layer, prompts in chunks -- against the
64-bit forward pass and against itself.

Keys, values and queries are rounded to f16 (half a step: 2^-11) once per layer.
That moves attention's output by at most 2^-11 (values) + 2 S 2^-11 (scores of
size S: two rounded factors each) of its weighted values, and each layer adds
such an error to the residual stream, whose norm it is a part of; S stays below 3
in these models, so logits are off by less than L (1 + 6) 2^-11 of their norm
(GEMVs: 1e-5)."""
import numpy as np
import pytest

import decode
from qwen2_numpy import Qwen2Numpy

pytestmark = pytest.mark.gpu

TINY = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000, rope_theta=1e6,
            norm_eps=1e-6, seed=7)
WIDE = dict(TINY, hidden=384, n_heads=6, n_kv_heads=1, head_dim=96, ffn=768, n_layers=3, seed=9)


def bound(cfg):
    return cfg["n_layers"] * 7 * 2.0 ** -11


def off(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def generate(m, prompt, n_gen):
    toks, _ = m.generate(prompt, n_gen)
    return toks, m.last_logits()


@pytest.mark.parametrize("cfg", [TINY, WIDE], ids=["tiny", "wide"])
@pytest.mark.parametrize("n_prompt", [1, 2, 17, 64, 65, 150])
def test_prompts_against_64_bits(oracle, cfg, n_prompt):
    with decode.Model(threads=8, **cfg) as m:
        p = decode.prompt_tokens(n_prompt, cfg["vocab"], n_prompt)
        _, ref = Qwen2Numpy(m, oracle).generate(p, 1)
        m.attach_gpu(0)
        m.set_attention(m.ATTENTION_GPU)
        _, got = generate(m, p, 1)
    assert off(got, ref) <= bound(cfg)


@pytest.mark.parametrize("cfg", [TINY, WIDE], ids=["tiny", "wide"])
def test_generated_tokens_continue_the_chunk(cfg):
    """A prompt in one chunk, the same tokens as a shorter prompt and forced
    ones: generation on n tokens gives the logits that a prompt of them gives."""
    with decode.Model(threads=8, **cfg) as m:
        m.attach_gpu(0)
        m.set_attention(m.ATTENTION_GPU)
        p = decode.prompt_tokens(30, cfg["vocab"], 4)
        toks, logits = generate(m, p, 40)
        _, again = generate(m, np.concatenate([p, toks[:39]]), 1)
        assert off(logits, again) <= bound(cfg)
        assert m.last_wait() == m.WAIT_FENCE
        same, same_logits = generate(m, p, 40)
        assert np.array_equal(same, toks) and np.array_equal(same_logits, logits)


def test_long_prompt_in_several_chunks():
    with decode.Model(threads=8, **TINY) as m:
        m.attach_gpu(0)
        p = decode.prompt_tokens(1100, 1000, 3)
        host, host_logits = generate(m, p, 1)
        m.set_attention(m.ATTENTION_GPU)
        m.set_wait(m.WAIT_STREAM)
        toks, logits = generate(m, p, 1)
        assert off(logits, host_logits) <= bound(TINY)
        assert m.last_wait() == m.WAIT_STREAM
        m.set_attention(m.ATTENTION_HOST)
        _, back = generate(m, p[:50], 2)
        assert m.last_wait() == m.WAIT_STREAM and np.all(np.isfinite(back))


def test_3b_layer_shapes():
    cfg = dict(decode.QWEN25_3B, n_layers=2)
    with decode.Model(threads=8, **cfg) as m:
        m.attach_gpu(0)
        p = decode.prompt_tokens(80, cfg["vocab"], 5)
        _, host = generate(m, p, 3)
        m.set_attention(m.ATTENTION_GPU)
        _, got = generate(m, p, 3)
    assert off(got, host) <= bound(cfg)
