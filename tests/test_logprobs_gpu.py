"""mi355x_logprobs against 64 bits.

Top tokens are equal.  Bounds of the rest, with u = 2^-24 and d = scale (max - x)
formed by two roundings (2 u d): an exponential has the relative error of its
argument's and a rounding (3 d u + 4 u), so S = sum exp(-d) has (3 E[d] + 4) u and a
sum's of V / 256 + 64 terms one behind the other; log S that much absolutely and half a
step; log p = -d - log S another 2 u d and a half step.  The entropy's second sum
has E[d] times the same and E[3 d^2] for the exponentials' errors."""
import numpy as np
import pytest

import layer_ref
import mi355x
from layer_ref import decode, encode
from mi355x import BF16, F16, F32

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ws(ctx):
    b = ctx.alloc(ctx.logprobs_workspace())
    mi355x.check(ctx.lib.mi355x_fill(ctx.h, b.ptr, 0, b.nbytes))
    yield b
    b.free()


class Logits:
    def __init__(self, ctx, ws, x, t=F32, top=5, tokens=None, scale=1.0, pad=0, shift=0, entropy=True, n_tokens=2,
                 seed=0):
        rng = np.random.default_rng([x.shape[1], seed])
        self.T, self.V = x.shape
        self.__dict__.update(ctx=ctx, t=t, top=top, scale=scale)
        raw = encode(x, t)
        self.x = decode(raw, t)
        self.stride = self.V + pad
        full = np.full((self.T, self.stride), encode(np.full(1, np.inf), t)[0])
        full[:, :self.V] = raw
        flat = np.concatenate([np.repeat(full[:1, -1], shift), full.reshape(-1)])
        self.tokens = rng.integers(0, self.V, (self.T, n_tokens)).astype(np.int32) if tokens is None else tokens
        k = self.tokens.shape[1]
        f = lambda n: ctx.to_device(np.full(n + 1, 7.0, np.float32))  # noqa: E731
        self.lx, self.tk = ctx.to_device(flat), ctx.to_device(self.tokens)
        self.lp, self.ent, self.tlp = f(self.T * k), f(self.T), f(self.T * top)
        self.tt = ctx.to_device(np.full(self.T * top + 1, 7, np.int32))
        self.args = mi355x.LogprobsArgs(n_rows=self.T, n_vocab=self.V, type=t,
                                        logits=self.lx.ptr + shift * raw.itemsize, stride=self.stride, scale=scale,
                                        n_tokens=k, tokens=self.tk.ptr, token_logprobs=self.lp.ptr,
                                        entropy=self.ent.ptr if entropy else None, n_top=top,
                                        top_tokens=self.tt.ptr, top_logprobs=self.tlp.ptr, workspace=ws.ptr,
                                        workspace_bytes=ws.nbytes)

    def verify(self):
        T, k, top, V = self.T, self.tokens.shape[1], self.top, self.V
        lp, ent = layer_ref.logprobs(self.x, self.scale)
        with np.errstate(invalid="ignore"):
            d = np.float64(np.float32(self.scale)) * (self.x.max(1, keepdims=True) - self.x)
        p = np.where(np.isfinite(lp), np.exp(np.where(np.isfinite(lp), lp, 0)), 0)
        d = np.where(p > 0, d, 0)
        mean, square = (p * d).sum(1), (p * d * d).sum(1)
        sums = (3 * mean + 4 + V / 256 + 64) * U

        def near(got, ref, bound, what):
            assert got[-1] == 7.0, what + ": behind the end"
            got = got[:-1].reshape(ref.shape).astype(np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(ref)), what
            assert np.array_equal(np.isinf(got), np.isinf(ref)), what
            ok = np.isfinite(ref)
            off = np.abs(got[ok] - ref[ok]) - np.broadcast_to(bound, ref.shape)[ok]
            assert not np.any(off > 0), (what, float(off.max()))

        tok = np.clip(self.tokens, 0, V - 1)
        ref = np.take_along_axis(lp, tok, 1)
        ref = np.where(tok == self.tokens, ref, np.nan)
        size = np.where(np.isfinite(ref), np.abs(ref), 0)
        near(self.lp.download(np.float32, T * k + 1), ref, sums[:, None] + 4 * U * size + U, "tokens")
        if self.args.entropy:
            bound = sums + (4 * mean + 3 * square) * U + mean * (sums + 4 * U) + U
            near(self.ent.download(np.float32, T + 1), ent, bound, "entropy")
        else:
            assert np.all(self.ent.download(np.float32, T + 1) == 7.0)
        if top:
            tt = self.tt.download(np.int32, T * top + 1)
            want = layer_ref.top_tokens(self.x, top)
            assert tt[-1] == 7 and np.array_equal(tt[:-1].reshape(T, top), want), \
                (np.argwhere(tt[:-1].reshape(T, top) != want)[:4], V)
            ref = np.where(want >= 0, np.take_along_axis(lp, np.maximum(want, 0), 1), -np.inf)
            ref[np.isnan(ent)] = np.nan
            size = np.where(np.isfinite(ref), np.abs(ref), 0)
            near(self.tlp.download(np.float32, T * top + 1), ref, sums[:, None] + 4 * U * size + U, "top")

    def free(self):
        for b in (self.lx, self.tk, self.lp, self.ent, self.tlp, self.tt):
            b.free()


def go(ctx, ws, *a, **kw):
    c = Logits(ctx, ws, *a, **kw)
    try:
        ctx.logprobs(c.args)
        ctx.sync()
        c.verify()
    finally:
        c.free()


def logits(T, V, seed=0, spread=2.5):
    rng = np.random.default_rng([T, V, seed])
    x = spread * rng.standard_normal((T, V))
    for r in range(T):
        x[r, rng.integers(0, V, 6)] += rng.uniform(4, 12)
    return x


@pytest.mark.parametrize("V", [1, 2, 7, 64, 65, 255, 256, 1000, 2047, 4096, 4100, 32003, 100001, 151936])
@pytest.mark.parametrize("t", [F32, BF16])
def test_vocabularies(ctx, ws, V, t):
    go(ctx, ws, logits(3, V), t, top=20)
    go(ctx, ws, logits(1, V), t, top=5)


@pytest.mark.parametrize("top", [0, 1, 2, 20, 63, 64])
@pytest.mark.parametrize("T,V", [(1, 30000), (1, 40), (5, 5000), (700, 1200)])
def test_top(ctx, ws, T, V, top):
    go(ctx, ws, logits(T, V, 1), F16, top=top)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (3, 5), (8, 8)])
def test_strides(ctx, ws, t, pad, shift):
    go(ctx, ws, logits(4, 9001, 2), t, pad=pad, shift=shift)
    go(ctx, ws, logits(1, 70001, 2), t, pad=pad, shift=shift)


@pytest.mark.parametrize("T", [2, 3, 17, 64, 255, 256, 257, 600, 2100])
def test_rows(ctx, ws, T):
    go(ctx, ws, logits(T, 3001, 3), BF16, top=7)


@pytest.mark.parametrize("scale", [0.25, 0.7, 1.25, 40.0, 1e-6])
def test_temperatures(ctx, ws, scale):
    go(ctx, ws, logits(3, 20000, 4), F32, scale=scale)
    go(ctx, ws, logits(1, 20000, 4), F32, scale=scale)


@pytest.mark.parametrize("T,V", [(6, 50), (6, 3000), (6, 60000), (1, 60000), (300, 5000)])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_equal_logits(ctx, ws, T, V, top):
    """Ties everywhere: rows of one value, of two, of few, of zeros of both signs."""
    rng = np.random.default_rng([V, top])
    x = rng.integers(0, 3, (T, V)).astype(np.float64)
    x[0] = 1.5
    if T > 1:
        x[1] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
        x[2] = rng.integers(-40, 1, V)
        x[3] = -x[2]
    go(ctx, ws, x, F32, top=top)
    go(ctx, ws, x, BF16, top=top)


@pytest.mark.parametrize("T", [1, 8])
@pytest.mark.parametrize("V", [500, 30000, 151936])
def test_orders(ctx, ws, T, V):
    """Rows that ascend, descend, have their largest side by side, or far apart in one thread's steps."""
    up = np.linspace(-20, 20, V)
    few = np.zeros(V)
    few[V // 3:V // 3 + 200] = 5 + np.arange(min(200, V - V // 3)) / 256
    steps = np.where(np.arange(V) % 2048 < 8, 3.0 + np.arange(V) / V, 0.0)
    nearly = np.where(np.arange(V) % 2048 < 152, 3.0 + np.arange(V) / V, 0.0)
    rows = [up, up[::-1], few, steps, nearly, -few, np.floor(up), np.floor(up)[::-1]]
    for x in rows if T == 1 else [None]:
        go(ctx, ws, np.stack(rows) if x is None else x[None], F32, top=20)
        go(ctx, ws, np.stack(rows) if x is None else x[None], F32, top=64)


@pytest.mark.parametrize("V", [40, 3000, 90000])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_masked_and_odd_logits(ctx, ws, V, t):
    """-inf in places, all but a few, everywhere; the type's lowest value; +inf and NaN."""
    rng = np.random.default_rng(V)
    x = logits(10, V, 5)
    low = {F32: -3.0e38, F16: -65504.0, BF16: -3.0e38}[t]
    x[1, rng.random(V) < 0.9] = -np.inf
    x[2] = -np.inf
    x[3] = -np.inf
    x[3, [V // 2, V - 1, 0]] = [1.0, 2.0, 1.0]
    x[4, rng.random(V) < 0.5] = low
    x[5] = low
    x[6, V - 1] = np.nan
    x[7, V // 2] = np.inf
    x[8], x[8, 3] = -np.inf, np.nan
    x[9] = -np.inf
    x[9, V // 3] = low
    tokens = rng.integers(0, V, (10, 4)).astype(np.int32)
    tokens[:, 0] = [-1, V, V // 2, 0, 2 ** 31 - 1, -2 ** 31, 0, 1, 3, V // 3]
    go(ctx, ws, x, t, top=20, tokens=tokens)
    for r in range(10):
        go(ctx, ws, x[r:r + 1], t, top=20, tokens=tokens[r:r + 1])


def test_large_logits(ctx, ws):
    """Differences that f32 holds, and rows that one token has nearly all of."""
    x = logits(4, 5000, 6)
    x[0] *= 1e4
    x[1] += 1e5
    x[2] *= 1e36
    x[3, 77] = 60
    go(ctx, ws, x, F32)
    for r in range(4):
        go(ctx, ws, x[r:r + 1], F32)


def test_what_is_not_asked_for(ctx, ws):
    x = logits(3, 4000, 7)
    go(ctx, ws, x, F32, top=0, entropy=False)
    go(ctx, ws, x, F32, top=3, entropy=False, n_tokens=0)
    go(ctx, ws, x, F32, top=0, n_tokens=300)
    go(ctx, ws, x[:1], F32, top=0, n_tokens=300)


def test_calls_share_a_workspace(ctx, ws):
    """Calls in order, without a wait between them; the counters are 0 again behind them."""
    cases = [Logits(ctx, ws, logits(T, V, 8), F32, top=top) for T, V, top in
             [(1, 151936, 20), (40, 20000, 5), (2, 60000, 64), (400, 3000, 1), (1, 5000, 0)]]
    try:
        for _ in range(3):
            for c in cases:
                ctx.logprobs(c.args)
        ctx.sync()
        for c in cases:
            c.verify()
        assert not ws.download(np.int32, 256).any()
    finally:
        for c in cases:
            c.free()


def test_rows_far_apart(ctx, ws):
    """Rows whose offsets pass 2^32 bytes."""
    x = logits(3, 6000, 9).astype(np.float32)
    stride = (1 << 30) + 4
    c = Logits(ctx, ws, x, F32)
    big = ctx.alloc(4 * (2 * stride + 6000))
    try:
        for r in range(3):
            big.upload(x[r], 4 * r * stride)
        c.args.logits, c.args.stride = big.ptr, stride
        ctx.logprobs(c.args)
        ctx.sync()
        c.verify()
    finally:
        big.free()
        c.free()


@pytest.mark.parametrize("V", [40, 2048, 9000, 40000])
@pytest.mark.parametrize("scale", [1.0, 0.75])
@pytest.mark.parametrize("t", [F32, BF16])
def test_rows_that_begin_with_the_lowest_value(ctx, ws, t, scale, V):
    """Sums against the lowest value, which a logit far above it then replaces: the
    difference's multiple passes f32's range."""
    x = logits(3, V, 8)
    low = float(decode(encode(np.full(1, np.finfo(np.float32).min if t == F32 else -3.3e38), t), t)[0])
    x[0, :V // 2] = low
    x[1, :V - 3] = low
    x[2, ::2] = low
    go(ctx, ws, x, t, scale=scale)
    for r in range(3):
        go(ctx, ws, x[r:r + 1], t, scale=scale)


def test_scales_at_their_limits(ctx, ws):
    x = logits(2, 5000, 9)
    go(ctx, ws, x * 2.0 ** 100, F32, scale=2.0 ** -100)
    go(ctx, ws, x * 2.0 ** -100, F32, scale=2.0 ** 100)


def test_more_rows_than_workgroups(ctx, ws):
    T = (1 << 20) + 77
    rng = np.random.default_rng(T)
    go(ctx, ws, 3 * rng.standard_normal((T, 9)), F16, top=2)
