"""mi355x_norm_q8 and mi355x_swiglu_q8 against 64 bits.

Codes are those of the 64-bit quotients: equal, but that a gate's value has the
64-bit rounding of an exponential (a few units of 2^-52 of a quotient of at most
127, 1e-12 at most), so that a quotient this near to a border may go either way.
Scales are rounded once: half a step of f32, and 1e-13 for the 64-bit sum, root
and exponential; below 2^-126 steps are 2^-149."""
import numpy as np
import pytest

import layer_ref
import mi355x
from layer_ref import decode, encode, storage
from mi355x import BF16, F16, F32

pytestmark = pytest.mark.gpu
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}


class Rows:
    """Rows of values of a type on the device, `stride` apart and `shift` values into the buffer."""

    def __init__(self, ctx, values, t, pad=0, shift=0):
        self.t, self.shape, self.shift = t, values.shape, shift
        self.stride = values.shape[1] + pad
        self.raw = encode(values, t)
        full = np.full((values.shape[0], self.stride), encode(np.full(1, 9.0), t)[0], storage(t))
        full[:, :values.shape[1]] = self.raw
        self.buf = ctx.to_device(np.concatenate([np.zeros(shift, storage(t)), full.reshape(-1)]))
        self.ptr = self.buf.ptr + shift * self.raw.itemsize
        self.values = decode(self.raw, t)

    def bits(self):
        """The rows now; what lies between them has not changed."""
        T, n = self.shape
        a = self.buf.download(storage(self.t), self.shift + T * self.stride)[self.shift:].reshape(T, self.stride)
        assert np.all(a[:, n:] == encode(np.full(1, 9.0), self.t)[0]), "between the rows"
        return a[:, :n]


class Codes:
    """Codes and scales of a call's rows, with room between and behind them."""

    def __init__(self, ctx, T, n, pad=0, shift=0):
        self.T, self.n, self.stride, self.shift = T, n, n + pad, shift
        self.q = ctx.to_device(np.full(shift + T * self.stride + 3, 85, np.int8))
        self.s = ctx.to_device(np.full(T + 1, 7.0, np.float32))
        self.ptr = self.q.ptr + shift

    def get(self):
        q = self.q.download(np.int8, self.shift + self.T * self.stride + 3)
        s = self.s.download(np.float32, self.T + 1)
        body = q[self.shift:-3].reshape(self.T, self.stride)
        assert np.all(q[:self.shift] == 85) and np.all(q[-3:] == 85) and np.all(body[:, self.n:] == 85), "outside"
        assert s[-1] == 7.0
        return body[:, :self.n], s[:-1]

    def free(self):
        self.q.free()
        self.s.free()


def check(got, ref, what):
    codes, scales = got
    want, scale, loose = ref
    wrong = (codes != want) & ~loose
    assert not wrong.any(), (what, np.argwhere(wrong)[:4], codes[wrong][:4], want[wrong][:4])
    assert np.all(np.abs(codes.astype(int) - want)[loose] <= 1)
    assert np.array_equal(np.isnan(scales), np.isnan(scale)), what
    ok = ~np.isnan(scale)
    with np.errstate(over="ignore"):
        past = np.abs(scale[ok]) > np.finfo(np.float32).max * (1 + 2.0 ** -25)
    assert np.all(np.isinf(scales[ok][past]))
    bound = scale[ok] * (2.0 ** -24 + 1e-13) + 2.0 ** -150
    assert np.all(np.abs(scales[ok].astype(np.float64) - scale[ok])[~past] <= bound[~past]), what


def values(T, n, seed, wide=True):
    rng = np.random.default_rng([T, n, seed])
    x = rng.standard_normal((T, n)) * np.exp(rng.standard_normal((T, 1)))
    if wide and n > 8:
        x[:, rng.integers(0, n, 2)] *= 30
    return x


def norm_case(ctx, T, n, t, res_t=None, norm=True, store=True, pad=0, shift=0, x=None, res=None, w=None, alias=None,
              eps=1e-6):
    rng = np.random.default_rng([n, T, 5])
    rx = Rows(ctx, values(T, n, 1) if x is None else x, t, pad, shift)
    rr = None
    if res_t is not None:
        rr = Rows(ctx, values(T, n, 2) if res is None else res, res_t, pad, shift)
    if norm and w is None:
        w = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
    wb = ctx.to_device(np.concatenate([np.zeros(shift % 2, np.float32), w])) if norm else None
    out = None
    if rr is not None and store:
        out = {"residual": rr, "x": rx}.get(alias) or Rows(ctx, np.zeros((T, n)), res_t, pad + 1, shift)
    c = Codes(ctx, T, n, pad, shift)
    try:
        ctx.norm_q8(mi355x.NormQ8Args(
            n_rows=T, n=n, type=t, x=rx.ptr, x_stride=rx.stride, residual_type=-1 if res_t is None else res_t, eps=eps,
            residual=rr.ptr if rr else None, residual_stride=rr.stride if rr else 0,
            residual_out=out.ptr if out else None, residual_out_stride=out.stride if out else 0,
            norm=wb.ptr + 4 * (shift % 2) if norm else None, q=c.ptr, q_stride=c.stride, scales=c.s.ptr))
        ctx.sync()
        h, t64, factor = layer_ref.norm_rows(rx.values, rr.values if rr else None, res_t, w if norm else None, eps)
        codes, scale, _ = layer_ref.codes_of(t64)
        bad = ~np.isfinite(t64).all(1)
        with np.errstate(invalid="ignore"):
            scale = np.where((scale == 0) & ~bad, 0, scale * factor)
        check(c.get(), (codes, scale, np.zeros(codes.shape, bool)), "norm")
        if out:
            assert np.array_equal(decode(out.bits(), res_t), h, equal_nan=True)
        if rr is not None and out is not rr:
            assert rr.bits().tobytes() == rr.raw.tobytes()
        if out is not rx:
            assert rx.bits().tobytes() == rx.raw.tobytes()
        return c.get()
    finally:
        for b in {id(r): r.buf for r in (rx, rr, out) if r}.values():
            b.free()
        if wb:
            wb.free()
        c.free()


SIZES = [1, 2, 7, 8, 9, 63, 64, 65, 100, 511, 512, 520, 1000, 2048, 4097, 5120, 8192, 8200, 16384, 16392, 24000, 32768,
         32769, 65528, 65536]


@pytest.mark.parametrize("n", SIZES)
def test_norm_sizes(ctx, n):
    norm_case(ctx, 3, n, BF16, BF16)


@pytest.mark.parametrize("res_t", [None, F32, F16, BF16])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,pad,shift", [(264, 0, 0), (331, 5, 3)])
def test_norm_types(ctx, t, res_t, n, pad, shift):
    for norm in (True, False):
        norm_case(ctx, 5, n, t, res_t, norm, pad=pad, shift=shift)


@pytest.mark.parametrize("n", [24, 777, 2048, 40000])
def test_norm_in_place(ctx, n):
    norm_case(ctx, 4, n, F16, F16, alias="residual", pad=3)
    norm_case(ctx, 4, n, F16, F16, alias="x", pad=3)
    norm_case(ctx, 4, n, BF16, F32, alias="residual")
    norm_case(ctx, 4, n, F32, F32, store=False)


@pytest.mark.parametrize("T", [1, 2, 255, 3000])
def test_norm_rows(ctx, T):
    norm_case(ctx, T, 96, BF16, F32)
    norm_case(ctx, T, 96, F32)


@pytest.mark.parametrize("n", [16, 600, 9000, 50000])
def test_norm_of_rows_without_a_scale(ctx, n):
    """Zeros; infinities, NaN, sums that the residual's type does not hold; the smallest and the largest values."""
    x = values(9, n, 3)
    x[0] = 0
    x[1, n // 2], x[2, 0], x[3, n - 1] = np.inf, -np.inf, np.nan
    x[4] = 1e-44 * np.sign(x[4])
    x[5] = 3e38 * np.sign(x[5])
    x[6] = 0
    x[6, n - 1] = 1e-30
    with np.errstate(over="ignore"):
        codes, scales = norm_case(ctx, 9, n, F32, x=x)
        assert scales[0] == 0 and np.isnan(scales[1:4]).all() and np.isfinite(scales[4:]).all()
        norm_case(ctx, 9, n, F32, norm=False, x=x)
        big = np.clip(x, -60000, 60000)
        codes, scales = norm_case(ctx, 9, n, F16, F16, x=big, res=big)
        assert np.isnan(scales[5])
        # a norm weight that is not finite, and one that takes a scale past f32
        w = np.ones(n, np.float32)
        w[1] = np.inf
        codes, scales = norm_case(ctx, 9, n, F32, x=x, w=w)
        assert np.isnan(scales).all()
        w[1] = 3e38
        norm_case(ctx, 9, n, F32, x=np.abs(values(9, n, 4)) + 1, w=w, eps=0.0)


def test_norm_ties_go_to_even(ctx):
    """Quotients of whole numbers and halves, with a largest value that 127 / max is not exact for."""
    k = np.arange(-127, 128)
    for unit in (1.0, 3.0, 5.0):
        x = np.concatenate([k, k[:-1] + 0.5]) * unit
        codes, scales = norm_case(ctx, 1, x.size, F32, norm=False, x=x[None])
        assert scales[0] == unit and np.array_equal(codes[0], np.rint(x / unit))


def swiglu_case(ctx, T, n, t, pad=0, shift=0, g=None, u=None, halves=False):
    g = values(T, n, 6, False) if g is None else g
    u = values(T, n, 7) if u is None else u
    if halves:
        both = Rows(ctx, np.concatenate([g, u], 1), t, pad, shift)
        bufs, strides = [both], (both.stride, both.stride)
        ptrs = both.ptr, both.ptr + n * both.raw.itemsize
        gv, uv = both.values[:, :n], both.values[:, n:]
    else:
        rg, ru = Rows(ctx, g, t, pad, shift), Rows(ctx, u, t, pad + 2, shift)
        bufs, strides, ptrs, gv, uv = [rg, ru], (rg.stride, ru.stride), (rg.ptr, ru.ptr), rg.values, ru.values
    c = Codes(ctx, T, n, pad, shift)
    try:
        ctx.swiglu_q8(mi355x.SwigluQ8Args(n_rows=T, n=n, type=t, gate=ptrs[0], gate_stride=strides[0], up=ptrs[1],
                                          up_stride=strides[1], q=c.ptr, q_stride=c.stride, scales=c.s.ptr))
        ctx.sync()
        check(c.get(), layer_ref.codes_of(layer_ref.swiglu(gv, uv), 1e-12), "swiglu")
        return c.get()
    finally:
        for b in bufs:
            b.buf.free()
        c.free()


@pytest.mark.parametrize("n", SIZES)
def test_swiglu_sizes(ctx, n):
    swiglu_case(ctx, 3, n, BF16, halves=True)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,pad,shift,halves", [(264, 0, 0, True), (331, 5, 3, False), (331, 0, 1, True)])
def test_swiglu_types(ctx, t, n, pad, shift, halves):
    swiglu_case(ctx, 5, n, t, pad, shift, halves=halves)


@pytest.mark.parametrize("T", [1, 2, 255, 3000])
def test_swiglu_rows(ctx, T):
    swiglu_case(ctx, T, 96, F32)


@pytest.mark.parametrize("n", [16, 600, 9000, 50000])
def test_swiglu_over_the_range(ctx, n):
    """Gates far to either side, small and large factors, infinities and NaN."""
    rng = np.random.default_rng(n)
    g, u = 40 * rng.standard_normal((12, n)), rng.standard_normal((12, n))
    g[1], g[2] = -np.abs(g[1]) * 3, np.abs(g[2]) * 3      # closed, and open
    u[3] *= 1e30
    g[3] *= 1e5
    u[4] *= 1e-38
    g[4] = -np.abs(g[4])
    g[5], u[5] = 0, 1e30
    g[6, n // 2], u[7, 0], g[8, n - 1], u[9, 1] = np.inf, -np.inf, np.nan, np.nan
    g[10], u[10] = 3e38, 3e38 * np.sign(u[10])            # products past f32
    g[11], u[11] = -rng.uniform(20, 100, n), np.exp(rng.uniform(20, 80, n))  # closed gates that large factors meet
    codes, scales = swiglu_case(ctx, 12, n, F32, g=g, u=u)
    assert np.isnan(scales[6:10]).all() and not codes[6:10].any() and scales[5] == 0 and np.isinf(scales[10])
    swiglu_case(ctx, 12, n, F16, g=np.clip(g, -6e4, 6e4), u=np.clip(u, -6e4, 6e4))
    with np.errstate(over="ignore"):
        swiglu_case(ctx, 12, n, BF16, g=g, u=u)


def test_rows_far_apart(ctx):
    """Rows whose offsets pass 2^32 bytes."""
    n, stride = 520, (1 << 30) + 264
    rng = np.random.default_rng(8)
    x = rng.standard_normal((3, n)).astype(np.float32)
    far = ctx.alloc(4 * (2 * stride + 2 * n))
    c = Codes(ctx, 3, n)
    try:
        for r in range(3):
            far.upload(x[r], 4 * r * stride)
            far.upload(x[2 - r], 4 * (r * stride + n))
        ctx.norm_q8(mi355x.NormQ8Args(n_rows=3, n=n, type=F32, x=far.ptr, x_stride=stride, residual_type=F32,
                                      residual=far.ptr + 4 * n, residual_stride=stride, residual_out=far.ptr + 4 * n,
                                      residual_out_stride=stride, q=c.ptr, q_stride=n, scales=c.s.ptr))
        ctx.sync()
        h = x + x[::-1]
        check(c.get(), layer_ref.codes_of(h.astype(np.float64)), "norm")
        for r in range(3):
            assert np.array_equal(far.download(np.float32, n, 4 * (r * stride + n)), h[r])
        ctx.swiglu_q8(mi355x.SwigluQ8Args(n_rows=3, n=n, type=F32, gate=far.ptr, gate_stride=stride,
                                          up=far.ptr + 4 * n, up_stride=stride, q=c.ptr, q_stride=n, scales=c.s.ptr))
        ctx.sync()
        check(c.get(), layer_ref.codes_of(layer_ref.swiglu(x.astype(np.float64), h.astype(np.float64)), 1e-12), "gate")
    finally:
        far.free()
        c.free()


@pytest.mark.parametrize("n", [64, 2048, 9000, 20000])
def test_swiglu_closed_gates_that_large_factors_meet(ctx, n):
    """A few of them among ordinary values: products that are next to nothing, about as large
    as the rest, the row's largest, and of gates whose exponential leaves f32's range."""
    rng = np.random.default_rng([n, 3])
    g, u = rng.standard_normal((8, n)), rng.standard_normal((8, n))
    at = rng.integers(0, n, 5)
    for r, (gate, factor) in enumerate([(-30, 1e12), (-30, 1e14), (-60, 1e25), (-86, 1e37), (-95, 3e38), (-9, 2e3),
                                        (-1e4, 3e38), (-20, 300)]):
        g[r, at] = gate * rng.uniform(0.99, 1.01, 5)
        u[r, at] = factor * rng.uniform(0.5, 1, 5)
    swiglu_case(ctx, 8, n, F32, g=g, u=u)
    swiglu_case(ctx, 8, n, BF16, g=g, u=u)
    swiglu_case(ctx, 8, n, F16, g=np.clip(g, -6e4, 6e4), u=np.clip(u, -6e4, 6e4))


@pytest.mark.parametrize("T", [256, 1025, 2500])
@pytest.mark.parametrize("n", [2048, 2059, 4099, 6000])
def test_many_rows_of_several_runs_a_thread(ctx, T, n):
    """Workgroups that go through several rows, and rows that end inside a thread's runs."""
    norm_case(ctx, T, n, BF16, BF16)
    norm_case(ctx, T, n, F16, F32, alias="residual", pad=1)
    norm_case(ctx, T, n, BF16, BF16, norm=False, alias="x")
    swiglu_case(ctx, T, n, BF16, halves=True)
    swiglu_case(ctx, T, n, F32, pad=3, shift=1)


def test_infinities_among_many_rows(ctx):
    """Rows that are not finite, or zero, between others that the same workgroup computes."""
    x = values(2100, 4100, 5)
    x[::7, 4099], x[1::7, 0], x[2::7] = np.inf, np.nan, 0
    norm_case(ctx, 2100, 4100, F32, F32, x=x, res=np.zeros_like(x))
    norm_case(ctx, 2100, 4100, BF16, x=x)
    g, u = values(2100, 4100, 6, False), x
    swiglu_case(ctx, 2100, 4100, F32, g=g, u=u)


def test_more_rows_than_workgroups(ctx):
    norm_case(ctx, (1 << 20) + 77, 9, BF16, BF16)
    swiglu_case(ctx, (1 << 20) + 77, 9, BF16)
