"""mi355x_qk_norm_rope against 64 bits.

Bound of a value: one rounding to the output type (half a step of the value),
and f32 arithmetic: the bias and the norm's two products and its factor (a sum
of at most 1024 squares by 64 lanes, a division and a root: 24 half steps of
2^-24 together), the sine and cosine (4 units: 2^-21 and the reduction of the
angle to a fraction of a turn in f32: half a step of at most half a turn, pi
2^-24), two products and a sum: 48 half steps of |a| + |b| in all."""
import numpy as np
import pytest

import mi355x
import paged_ref
from mi355x import BF16, F16, F32
from paged_ref import HALF_STEP, decode, encode, storage

pytestmark = pytest.mark.gpu


def check(got, ref, size, t, what):
    # subnormal results of f16 are steps of 2^-24
    bound = HALF_STEP[t] * np.abs(ref) + 48 * 2.0 ** -24 * size + (2.0 ** -25 if t == F16 else 0)
    off = np.abs(got - ref) - bound
    assert np.all(off <= 0), (what, float(off.max()))


class Case:
    def __init__(self, ctx, T, hq, hk, hd, rot, pairs, tin, tout, bias, norm, pool=True, page=16, hnd=False, gap=0,
                 pad=0, pos=5000, seed=0, spare=2, shift=0):
        rng = np.random.default_rng([seed, T, hd])
        self.__dict__.update(ctx=ctx, T=T, hq=hq, hk=hk, hd=hd, rot=rot, pairs=pairs, tin=tin, tout=tout)
        width = (hq + 2 * hk) * hd + pad
        self.width, self.shift = width, shift
        self.raw = encode(1.5 * rng.standard_normal((T, width)), tin)
        x = decode(self.raw, tin)
        self.q, self.k, self.v = (x[:, a * hd:b * hd].reshape(T, -1, hd)
                                  for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
        f32 = lambda n: rng.standard_normal(n).astype(np.float32)  # noqa: E731
        self.bias = [f32(h * hd) for h in (hq, hk, hk)] if bias else [None] * 3
        self.norm = [(1 + 0.3 * f32(hd)) for _ in range(2)] if norm else [None] * 2
        self.positions = rng.integers(0, pos, T).astype(np.int32)
        self.inv_freq = (1e6 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32)
        self.pool = None
        es = encode(np.zeros(1), tin).itemsize
        head = np.zeros(shift, storage(tin))  # rows that start `shift` values into the buffer
        self.inb = ctx.to_device(np.concatenate([head, self.raw.reshape(-1)]))
        base = self.inb.ptr + shift * es
        self.qs = hq * hd + 8
        self.bufs = [self.inb]
        self.qout = self.dev(encode(np.full((T, self.qs), 7.0), tout))
        ptr = lambda a: self.dev(a).ptr if a is not None else None  # noqa: E731
        kw = dict(n_rows=T, n_heads=hq, n_kv_heads=hk, head_dim=hd, rot_dim=rot,
                  rope_mode=mi355x.ROPE_PAIRS if pairs else mi355x.ROPE_HALVES, in_type=tin, out_type=tout, eps=1e-6,
                  q=base, k=base + hq * hd * es, v=base + (hq + hk) * hd * es, q_stride=width, k_stride=width,
                  v_stride=width, q_bias=ptr(self.bias[0]), k_bias=ptr(self.bias[1]), v_bias=ptr(self.bias[2]),
                  q_norm=ptr(self.norm[0]), k_norm=ptr(self.norm[1]), positions=ptr(self.positions),
                  inv_freq=ptr(self.inv_freq) if rot else None, q_out=self.qout.ptr, q_out_stride=self.qs)
        if pool:
            n_pages = -(-T // page) + spare
            self.pool = paged_ref.Pool(ctx, rng, tout, n_pages, page, hk, hd, hnd, gap)
            self.slots = rng.permutation(n_pages * page)[:T].astype(np.int64)
            self.struct = self.pool.struct()
            kw.update(pool=mi355x.pointer(self.struct), slots=ptr(self.slots))
        else:
            self.kout = self.dev(encode(np.full((T, hk * hd), 7.0), tout))
            kw.update(k_out=self.kout.ptr, k_out_stride=hk * hd)
        self.args = mi355x.QkNormRopeArgs(**kw)

    def dev(self, a):
        self.bufs.append(self.ctx.to_device(a))
        return self.bufs[-1]

    def refs(self):
        f = lambda x, b, n, r: paged_ref.rope(x, b, n, 1e-6, self.positions, self.inv_freq, r, self.pairs)  # noqa: E731
        return (f(self.q, self.bias[0], self.norm[0], self.rot), f(self.k, self.bias[1], self.norm[1], self.rot),
                f(self.v, self.bias[2], None, 0))

    def queries(self):
        q = decode(self.qout.download(storage(self.tout), self.T * self.qs), self.tout).reshape(self.T, self.qs)
        w = self.hq * self.hd
        assert np.all(q[:, w:] == 7.0), "between the rows"
        return q[:, :w].reshape(self.T, self.hq, self.hd)

    def verify(self, stored=None):
        rq, rk, rv = self.refs()
        check(self.queries(), *rq, self.tout, "q")
        if self.pool is None:
            k = decode(self.kout.download(storage(self.tout), self.T * self.hk * self.hd), self.tout)
            check(k.reshape(self.T, self.hk, self.hd), *rk, self.tout, "k")
            return
        rows = np.arange(self.T) if stored is None else stored
        pg, at = self.slots[rows] // self.pool.page, self.slots[rows] % self.pool.page
        for name, got, old, (ref, size) in zip("kv", self.pool.download(), (self.pool.k, self.pool.v), (rk, rv)):
            check(got[pg, at], ref[rows], size[rows], self.tout, name)
            rest = np.ones(old.shape[:2], bool)
            rest[pg, at] = False
            assert np.array_equal(got[rest], old[rest]), name + ": other slots"

    def free(self):
        for b in self.bufs:
            b.free()
        if self.pool:
            self.pool.free()


def go(ctx, *a, **kw):
    c = Case(ctx, *a, **kw)
    try:
        ctx.qk_norm_rope(c.args)
        ctx.sync()
        c.verify()
    finally:
        c.free()


@pytest.mark.parametrize("tin,tout", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, BF16)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("T,hq,hk,hd,rot,bias,norm", [
    (1, 16, 2, 128, 128, True, False), (7, 14, 2, 64, 64, True, True), (33, 8, 8, 96, 96, False, True),
    (130, 4, 1, 256, 128, False, False), (1, 3, 1, 8, 8, True, True), (5, 2, 2, 512, 512, False, True),
    (600, 32, 8, 128, 128, False, True)])
def test_types_and_sizes(ctx, T, hq, hk, hd, rot, bias, norm, pairs, tin, tout):
    go(ctx, T, hq, hk, hd, rot, pairs, tin, tout, bias, norm)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("hd,rot", [(80, 80), (128, 6), (40, 20), (1024, 1000), (64, 0), (72, 36), (24, 16)])
def test_odd_heads_and_partial_rotations(ctx, hd, rot, pairs):
    go(ctx, 9, 3, 2, hd, rot, pairs, F32, F16, True, True)


@pytest.mark.parametrize("kw", [dict(hnd=True, page=8), dict(gap=8, page=1), dict(hnd=True, gap=16, page=64),
                                dict(pad=5), dict(pad=8, shift=3), dict(page=256)])
def test_strides_and_alignments(ctx, kw):
    for tin in (F32, BF16):
        go(ctx, 21, 6, 2, 64, 64, False, tin, BF16, True, True, **kw)


@pytest.mark.parametrize("tout", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [6, 64, 128])
def test_without_a_pool(ctx, hd, tout):
    go(ctx, 19, 4, 2, hd, hd, False, F32, tout, True, True, pool=False)


def test_far_positions(ctx):
    go(ctx, 64, 2, 1, 128, 128, False, F32, F16, False, False, pos=2 ** 31 - 1)


def test_rows_without_a_slot_store_nothing(ctx):
    c = Case(ctx, 12, 4, 2, 64, 64, False, F32, F16, True, True, page=4)
    try:
        bad = np.array([0, 5, 11])
        c.slots[bad] = [-1, c.pool.n_pages * 4, -2 ** 40]
        c.slots[6] = 2 ** 62
        buf = ctx.to_device(c.slots)
        c.args.slots = buf.ptr
        ctx.qk_norm_rope(c.args)
        ctx.sync()
        c.verify(stored=np.array([1, 2, 3, 4, 7, 8, 9, 10]))
        buf.free()
    finally:
        c.free()


@pytest.mark.parametrize("t,hd", [(F32, 64), (F16, 128), (BF16, 20)])
def test_queries_and_keys_in_place(ctx, t, hd):
    c = Case(ctx, 10, 4, 2, hd, hd, False, t, t, True, True, pool=False)
    try:
        c.args.q_out, c.args.q_out_stride = c.args.q, c.args.q_stride
        c.args.k_out, c.args.k_out_stride = c.args.k, c.args.k_stride
        ctx.qk_norm_rope(c.args)
        ctx.sync()
        got = decode(c.inb.download(storage(t), c.raw.size), t).reshape(c.T, c.width)
        rq, rk, _ = c.refs()
        check(got[:, :4 * hd].reshape(10, 4, hd), *rq, t, "q")
        check(got[:, 4 * hd:6 * hd].reshape(10, 2, hd), *rk, t, "k")
        assert np.array_equal(got[:, 6 * hd:], decode(c.raw, t)[:, 6 * hd:])
    finally:
        c.free()


def test_zero_rows_of_a_norm_and_non_finite_values(ctx):
    """A head of zeros stays zero (eps), and one head's NaN stays its own."""
    c = Case(ctx, 3, 4, 2, 64, 64, False, F32, F16, False, True)
    try:
        raw = c.raw.copy()
        raw[0, :64] = 0.0
        raw[1, 64:128] = np.nan
        c.inb.upload(raw)
        ctx.qk_norm_rope(c.args)
        ctx.sync()
        q = c.queries()
        assert np.all(q[0, 0] == 0) and np.all(np.isnan(q[1, 1]))
        q[0, 0], q[1, 1] = 1.0, 1.0
        assert np.all(np.isfinite(q))
    finally:
        c.free()


def test_more_rows_than_workgroups(ctx):
    """Past 2^22 rows a workgroup takes several: the first and the last ones."""
    T, hd = 2 ** 22 + 2 ** 20 + 3, 8
    rng = np.random.default_rng(5)
    x = rng.standard_normal((T, hd), dtype=np.float32)
    pos = np.arange(T, dtype=np.int32)
    freq = (1e4 ** (-2.0 * np.arange(hd // 2) / hd)).astype(np.float32)
    bufs = [ctx.to_device(a) for a in (x, pos, freq, np.zeros(T * hd, np.float32))]
    try:
        ctx.qk_norm_rope(mi355x.QkNormRopeArgs(
            n_rows=T, n_heads=1, n_kv_heads=0, head_dim=hd, rot_dim=hd, rope_mode=mi355x.ROPE_HALVES, in_type=F32,
            out_type=F32, eps=1e-6, q=bufs[0].ptr, q_stride=hd, positions=bufs[1].ptr, inv_freq=bufs[2].ptr,
            q_out=bufs[3].ptr, q_out_stride=hd))
        ctx.sync()
        got = bufs[3].download(np.float32, T * hd).reshape(T, 1, hd)
        for part in (slice(0, 5000), slice(T // 2, T // 2 + 5000), slice(T - 5000, T)):
            check(got[part], *paged_ref.rope(x[part, None], None, None, 1e-6, pos[part], freq, hd, False), F32, part)
    finally:
        for b in bufs:
            b.free()
