"""A row's attention does not depend on tokens that it does not see, down to the
last bit: finite keys of any size there, which move the maxima of other rows of the
same block, leave it as it was."""
import numpy as np
import pytest

from mi355x import BF16, F16, F32
from paged_ref import decode, encode
from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("q_lens,kv,hq,hk,hd", [
    ([3], [300], 4, 2, 64), ([4], [30000], 4, 1, 64), ([4, 2, 1], [9000, 333, 7000], 4, 1, 128), ([60], [300], 4, 2, 64), ([60, 2, 33], [700, 300, 90], 8, 2, 96),
    ([1100], [1400], 2, 1, 128), ([40], [500], 4, 1, 256)])
@pytest.mark.parametrize("window", [0, 250])
def test_large_keys_behind_a_row_leave_it_as_it_was(ctx, q_lens, kv, hq, hk, hd, window, t, out):
    c = Case(ctx, q_lens, kv, hq, hk, hd, t, out, window=window)
    try:
        clean = c.run().outputs()
        c.verify()
        last = c.offsets[1:] - 1
        group = hq // hk
        for s, k in enumerate(kv):  # the last token's key, which its own row alone sees, eight times its query
            at = c.table[s][(k - 1) // 16], (k - 1) % 16
            c.pool.k[at] = decode(encode(8.0 * c.q[last[s], ::group], t), t)
        c.pool.upload()
        c.struct.k, c.struct.v = (b.ptr for b in c.pool.bufs)
        got = c.run().outputs()
        c.verify()
        rest = np.setdiff1d(np.arange(c.offsets[-1]), last)
        assert np.array_equal(got[rest], clean[rest])
        assert not np.array_equal(got[last], clean[last])
    finally:
        c.free()
