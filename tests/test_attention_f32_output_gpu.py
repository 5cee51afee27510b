"""Attention with f32 output is as exact as f32, whatever the pages' 16-bit type.

Two tokens: the first has score 0 and value 0, the second score s <= 0 and value 1,
so that the output is w / (1 + w), w = e^s.  One value of q and k alone is not zero, so
q . k is exact, and what is left is f32 roundings, in units of 2^-24 of w: the scale, its
product with log2 e and the score's with that (3 of the exponent, which is |s| log2 e <=
5.8, each times ln 2: 12.1), the subtraction of the reference (up to 8 above and 7 below
it: half a step of a value below 16 is 2^3 ln 2 = 5.6, twice where the raise is apart),
the exponential (1 unit, 2), the sum, the reciprocal (1 unit, 2) and the product with it
(4 in all), and the joins of wavefronts and parts (exact: the others have no weight).
Together 30.  The weights' planes may add one such rounding."""
import numpy as np
import pytest

from mi355x import BF16, F16, F32
from paged_ref import decode, encode
from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("q_lens", [[1] * 40, [60, 30]])
@pytest.mark.parametrize("hq,hk,hd", [(8, 2, 64), (4, 1, 96), (16, 16, 128), (4, 1, 256)])
def test_weights_of_two_tokens(ctx, hq, hk, hd, q_lens, t):
    c = Case(ctx, q_lens, [2] * len(q_lens), hq, hk, hd, t, F32, causal=False)
    try:
        c.scale = c.args.scale = 0.125
        c.q[:] = 0.0
        c.q[..., 3] = decode(encode(-32.0 * c.rng.random(c.q.shape[:2]), t), t)
        for s in range(len(q_lens)):
            p = c.table[s, 0]
            c.pool.k[p, :2], c.pool.v[p, :2] = 0.0, 0.0
            c.pool.k[p, 1, :, 3], c.pool.v[p, 1] = 1.0, 1.0
        c.pool.upload()
        c.struct.k, c.struct.v = (b.ptr for b in c.pool.bufs)
        c.upload()
        got = c.run().outputs()
        w = np.exp(c.q[..., 3:4] * 0.125)
        off = np.abs(got / (w / (1 + w)) - 1)
        assert off.max() <= 31 * 2.0 ** -24, float(off.max() * 2 ** 24)
    finally:
        c.free()
