"""The decode harness with attention on the GPU fails a generation whose plan of pages
was refused (its later passes write and read nothing then), and recovers."""
import numpy as np
import pytest

import decode
import mi355x

pytestmark = pytest.mark.gpu

TINY = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000, rope_theta=1e6,
            norm_eps=1e-6, seed=7)


@pytest.mark.parametrize("wait", [decode.Model.WAIT_FENCE, decode.Model.WAIT_STREAM])
@pytest.mark.parametrize("skip", [0, 1, 5])  # the prompt's pass, the first token's, a later one's
def test_a_refused_plan_fails_the_generation(skip, wait):
    with decode.Model(threads=4, **TINY) as m:
        m.attach_gpu(0)
        m.set_wait(wait)
        m.set_attention(m.ATTENTION_GPU)
        p = decode.prompt_tokens(20, 1000, 1)
        toks, _ = m.generate(p, 8)
        mi355x.inject_fault("mi355x_kv_plan_pages", mi355x.HIP_ERROR_OUT_OF_MEMORY, skip)
        try:
            with pytest.raises(RuntimeError, match=f"no place.*status {mi355x.KV_PAGES}"):
                m.generate(p, 8)
        finally:
            mi355x.inject_fault(None)
        again, _ = m.generate(p, 8)
        assert np.array_equal(again, toks)


def test_a_refused_plan_of_the_operator(ctx):
    """The same refusal of one call: nothing taken, and the next one as if it had not been."""
    d = ctx.to_device
    i32 = lambda v: d(np.asarray(v, np.int32))  # noqa: E731
    b = dict(cached=i32([4]), added=i32([2]), block_table=i32([7, -1]), free_pages=i32([3, 5]), free_head=i32([0]),
             free_head_out=i32([-9]), row_offsets=i32([-9, -9]), kv_lens=i32([-9]), positions=i32([-9, -9]),
             slots=d(np.full(2, -9, np.int64)), status=i32([-9]))
    args = mi355x.KvPlanArgs(n_seqs=1, page_tokens=4, table_cols=2, n_free=2, table_stride=2, n_rows=2,
                             **{k: v.ptr for k, v in b.items()})
    try:
        mi355x.inject_fault("mi355x_kv_plan_pages", mi355x.HIP_ERROR_OUT_OF_MEMORY)
        ctx.kv_plan(args)
        ctx.sync()
        got = {k: list(b[k].download(np.int64 if k == "slots" else np.int32, n))
               for k, n in dict(status=1, free_head_out=1, row_offsets=2, block_table=2, slots=2).items()}
        assert got == dict(status=[mi355x.KV_PAGES], free_head_out=[0], row_offsets=[0, 0], block_table=[7, -1],
                           slots=[-1, -1])
        ctx.kv_plan(args)
        ctx.sync()
        assert list(b["status"].download(np.int32, 1)) == [0] and list(b["slots"].download(np.int64, 2)) == [12, 13]
    finally:
        mi355x.inject_fault(None)
        for v in b.values():
            v.free()
