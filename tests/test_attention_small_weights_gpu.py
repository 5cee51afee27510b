"""One token that takes nearly all of a row's weight and whose values are zero: the
output is what the others, far below it, add up to.  Many requests share the pages, so
that a workgroup meets that token and many others in one go.

Bound of a value, with weights w_j, A = sum_j w_j |v_j|, S the largest sum
scale |q_d k_jd| and n tokens.  As for any attention here: half a step of the output; the
weights' half step (2^-11, 2^-8) times A, or its square where they go in as two planes;
2 (hd + 8) S + n + 16 f32 roundings of A.  For f16 besides: a weight is held in steps of
2^-24 where the largest one of its tile (64 tokens at most) lies between 2^-1 and 2^15,
so that it is off by at most half a step, 2^-24 of that largest one, and rounds to
nothing at worst: min(2^-24 w_top, w_j) |v_j|."""
import numpy as np
import pytest

from mi355x import BF16, F16, F32
from paged_ref import HALF_STEP, decode, encode
from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu

KINDS = [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]


class Shared:
    """`copies` requests of q new tokens on the same kv tokens, all queries 1: scores are
    sums of a key's values times the scale, N(0, 1) of random keys.  Values are not
    negative, so that nothing cancels."""

    def __init__(self, ctx, copies, q, kv, hq, hk, hd, t, out, softcap=0.0):
        self.c = c = Case(ctx, [q] * copies, [kv] + [0] * (copies - 1), hq, hk, hd, t, out, page=64, softcap=softcap)
        self.q, self.n, self.copies = q, kv, copies
        c.kv[:] = kv
        c.table[:] = c.table[0]
        c.q[:] = 1.0
        c.pool.v = np.abs(c.pool.v)

    def at(self, j):
        return self.c.table[0][j // 64], j % 64

    def key(self, j, score):
        """Token j's key, such that its score is as given (about, in 16 bits)."""
        c = self.c
        c.pool.k[self.at(j)] = decode(encode(np.full((c.hk, c.hd), score / (c.hd * c.scale)), c.t), c.t)

    def verify(self, two_planes):
        c = self.c
        c.pool.upload()
        c.struct.k, c.struct.v = (b.ptr for b in c.pool.bufs)
        c.upload()
        got = c.run().outputs().reshape(self.copies, self.q, c.hq, c.hd)
        j = np.arange(self.n)
        k, v = (x[c.table[0][j // 64], j % 64] for x in (c.pool.k, c.pool.v))
        half = HALF_STEP[c.t]
        for h in range(c.hq):
            s = c.scale * k[:, h * c.hk // c.hq].sum(1)
            size = np.abs(c.scale) * np.abs(k[:, h * c.hk // c.hq]).sum(1).max()
            if c.softcap:
                s = c.softcap * np.tanh(s / c.softcap)
            seen = j <= self.n - self.q + np.arange(self.q)[:, None]
            w = np.where(seen, np.exp(s - s[:self.n - self.q + 1].max()), 0.0)
            w /= w.sum(1, keepdims=True)
            vh = v[:, h * c.hk // c.hq]
            ref, mag = w @ vh, w @ np.abs(vh)
            bound = HALF_STEP[c.out_t] * np.abs(ref)
            bound += ((half ** 2 if two_planes else half) + 2.0 ** -24 * (2 * (c.hd + 8) * size + self.n + 16)) * mag
            if c.t == F16:
                tops = np.maximum.reduceat(w, np.arange(0, self.n, 64), axis=1)[:, j // 64]
                bound += np.minimum(2.0 ** -24 * tops, w) @ np.abs(vh)
            if c.out_t == F16:
                bound += 2.0 ** -25
            off = np.abs(got[:, :, h] - ref)
            assert np.all(off <= bound), (h, float((off / bound).max()))

    def free(self):
        self.c.free()


def run(ctx, copies, q, kv, hq, hk, hd, t, out, nats, where, two_planes, **kw):
    s = Shared(ctx, copies, q, kv, hq, hk, hd, t, out, **kw)
    try:
        j = int(where * (kv - q))  # every row sees it
        s.key(j, nats)
        s.c.pool.v[s.at(j)] = 0.0
        s.verify(two_planes)
    finally:
        s.free()


@pytest.mark.parametrize("t,out", KINDS)
@pytest.mark.parametrize("nats", [8, 12, 16, 18])
@pytest.mark.parametrize("where", [0.0, 0.4, 1.0])
def test_single_tokens(ctx, where, nats, t, out):
    run(ctx, 1000, 1, 8000, 4, 1, 64, t, out, nats, where, True)


@pytest.mark.parametrize("t,out", KINDS)
@pytest.mark.parametrize("nats", [8, 12, 16, 18])
@pytest.mark.parametrize("where", [0.0, 0.4, 1.0])
def test_chunks(ctx, where, nats, t, out):
    run(ctx, 300, 40, 8000, 4, 1, 64, t, out, nats, where, out == F32)


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("copies,q", [(700, 1), (300, 60)])
@pytest.mark.parametrize("hd", [96, 128, 256])
def test_heads(ctx, hd, copies, q, out):
    run(ctx, copies, q, 3000, 4, 1, hd, F16, out, 17, 0.0, q == 1 or out == F32)


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("copies,q", [(1000, 1), (300, 40)])
@pytest.mark.parametrize("cap", [24.0, 100.0])  # times log2 e below 64, and above
def test_under_a_cap(ctx, cap, copies, q, out):
    run(ctx, copies, q, 8000, 4, 1, 64, F16, out, 20, 0.1, q == 1 or out == F32, softcap=cap)


@pytest.mark.parametrize("q,hq,hk", [(2050, 2, 1), (1100, 32, 16)])
def test_a_prompt_whose_first_token_takes_the_weight(ctx, q, hq, hk):
    """Workgroups of 256 rows, their keys in parts (one KV head) and whole (sixteen)."""
    run(ctx, 1, q, q, hq, hk, 128, F16, F32, 18, 0.0, True)


@pytest.mark.parametrize("copies,q", [(1000, 1), (300, 40)])
def test_several_levels_of_weights(ctx, copies, q):
    """Tokens of falling scores, 10 nats from one to the next, alone with values that
    are not zero, each in its own."""
    s = Shared(ctx, copies, q, 2000, 4, 1, 64, F16, F32)
    try:
        s.c.pool.v[:] = 0.0
        for i in range(4):
            s.key(300 * i, 40 - 10 * i)
            s.c.pool.v[s.at(300 * i)][:, i] = 60000.0
        s.verify(True)
    finally:
        s.free()
