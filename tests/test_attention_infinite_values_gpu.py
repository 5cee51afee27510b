"""An infinite value of v that a row sees makes that value of its output infinite or
NaN, and no other: not its other values, and not the rows that do not see the token."""
import numpy as np
import pytest

from mi355x import BF16, F16, F32
from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("q_lens,kv,hq,hk,hd", [([1, 3], [300, 200], 4, 2, 64), ([60, 33], [300, 90], 4, 2, 64),
                                                ([1100], [1200], 2, 1, 96), ([40], [200], 4, 1, 256)])
@pytest.mark.parametrize("back", [0, 1, 70])
def test_an_infinite_value(ctx, q_lens, kv, hq, hk, hd, back, t, out):
    """`back` tokens before each request's last one."""
    c = Case(ctx, q_lens, kv, hq, hk, hd, t, out)
    try:
        clean = c.run().outputs()
        hit = np.zeros(clean.shape, bool)
        for s, k in enumerate(kv):
            j = k - 1 - back
            c.pool.v[c.table[s][j // 16], j % 16, hk - 1, 5 + s] = np.inf if s == 0 else -np.inf
            first = c.offsets[s + 1] - 1 - back  # the row at that position, if it is a new one
            hit[max(c.offsets[s], first):c.offsets[s + 1], (hk - 1) * hq // hk:, 5 + s] = True
        c.pool.upload()
        c.struct.k, c.struct.v = (b.ptr for b in c.pool.bufs)
        got = c.run().outputs()
        assert not np.any(np.isfinite(got[hit]))
        assert np.array_equal(got[~hit], clean[~hit])
    finally:
        c.free()
