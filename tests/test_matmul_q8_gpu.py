"""mi355x_matmul_q8 against whole numbers: the sum is exact, and the three f32
operations and the rounding behind it are the stated ones, so every bit is
equal."""
import numpy as np
import pytest

import layer_ref
import mi355x
from layer_ref import decode, encode, storage
from mi355x import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws(ctx):
    b = ctx.alloc(ctx.matmul_q8_workspace())
    mi355x.check(ctx.lib.mi355x_fill(ctx.h, b.ptr, 0, b.nbytes))
    yield b
    b.free()


class Product:
    def __init__(self, ctx, ws, M, N, K, t=F32, bias=False, xpad=0, wpad=0, opad=0, oshift=0, lo=-127, seed=0):
        rng = np.random.default_rng([M, N, K, seed])
        self.__dict__.update(ctx=ctx, M=M, N=N, K=K, t=t, ostride=N + opad, oshift=oshift)
        self.x = rng.integers(lo, 128, (M, K)).astype(np.int8)
        self.w = rng.integers(lo, 128, (N, K)).astype(np.int8)
        self.xs = np.exp(rng.standard_normal(M)).astype(np.float32) * np.float32(0.01)
        self.wsc = np.exp(rng.standard_normal(N)).astype(np.float32) * np.float32(0.001)
        self.b = rng.standard_normal(N).astype(np.float32) if bias else None
        xf, wf = np.full((M, K + xpad), 99, np.int8), np.full((N, K + wpad), 99, np.int8)
        xf[:, :K], wf[:, :K] = self.x, self.w
        # the last rows end with their codes
        dev = lambda a: ctx.to_device(a)  # noqa: E731
        self.bufs = [dev(xf.reshape(-1)[:(M - 1) * (K + xpad) + K]), dev(wf.reshape(-1)[:(N - 1) * (K + wpad) + K]),
                     dev(self.xs), dev(self.wsc), dev(self.b) if bias else None]
        self.out = dev(np.full(oshift + M * self.ostride + 3, encode(np.full(1, 7.0), t)[0], storage(t)))
        p = [b.ptr if b else None for b in self.bufs]
        self.args = mi355x.MatmulQ8Args(n_rows=M, n_out=N, k=K, x=p[0], x_stride=K + xpad, x_scales=p[2], w=p[1],
                                        w_stride=K + wpad, w_scales=p[3], bias=p[4],
                                        out=self.out.ptr + oshift * self.itemsize(), out_type=t,
                                        out_stride=self.ostride, workspace=ws.ptr, workspace_bytes=ws.nbytes)

    def itemsize(self):
        return np.dtype(storage(self.t)).itemsize

    def ref(self):
        return layer_ref.matmul(self.x, self.w, self.xs, self.wsc, self.b, self.t)

    def got(self):
        a = self.out.download(storage(self.t), self.oshift + self.M * self.ostride + 3)
        seven = encode(np.full(1, 7.0), self.t)[0]
        body = a[self.oshift:-3].reshape(self.M, self.ostride)
        assert np.all(a[:self.oshift] == seven) and np.all(a[-3:] == seven) and np.all(body[:, self.N:] == seven), \
            "outside the rows"
        return body[:, :self.N]

    def verify(self):
        got, ref = self.got(), self.ref()
        same = np.array_equal(got, ref) if self.t == BF16 else np.array_equal(got, ref, equal_nan=True)
        assert same, (self.M, self.N, self.K, np.argwhere(got != ref)[:5], got[got != ref][:5], ref[got != ref][:5])

    def free(self):
        for b in (*self.bufs, self.out):
            if b:
                b.free()


def go(ctx, ws, *a, **kw):
    c = Product(ctx, ws, *a, **kw)
    try:
        ctx.matmul_q8(c.args)
        ctx.sync()
        c.verify()
    finally:
        c.free()


@pytest.mark.parametrize("K", [16, 48, 64, 80, 128, 144, 256, 1040, 2048, 4112])
@pytest.mark.parametrize("M", [1, 2, 3, 8, 15, 16, 17, 31, 33, 64, 65, 100, 129, 257])
def test_rows_and_depths(ctx, ws, M, K):
    go(ctx, ws, M, 130, K)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 64, 65, 127, 129, 255, 257, 1000, 2049])
@pytest.mark.parametrize("M", [1, 5, 16, 40, 128, 300])
def test_channels(ctx, ws, M, N):
    go(ctx, ws, M, N, 320, BF16)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (7, 96, 4096), (48, 264, 1024), (200, 520, 768), (513, 770, 272)])
def test_types(ctx, ws, M, N, K, t, bias):
    go(ctx, ws, M, N, K, t, bias)


@pytest.mark.parametrize("M,N", [(1, 77), (9, 64), (70, 200), (300, 260)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_strides(ctx, ws, M, N, t):
    go(ctx, ws, M, N, 208, t, True, xpad=16, wpad=48, opad=5, oshift=1)
    go(ctx, ws, M, N, 256, t, False, xpad=128, wpad=16, opad=8, oshift=8)


@pytest.mark.parametrize("M,N,K", [(1, 40, 131056), (3, 17, 131056), (20, 33, 131056), (70, 130, 65552),
                                   (260, 300, 16400)])
def test_longest_rows_of_the_largest_codes(ctx, ws, M, N, K):
    """-128 times -128 throughout: the largest sum that 32 bits hold."""
    c = Product(ctx, ws, M, N, K)
    try:
        for buf, rows in ((c.bufs[0], M), (c.bufs[1], N)):
            mi355x.check(ctx.lib.mi355x_fill(ctx.h, buf.ptr, 0x80, buf.nbytes))
        c.x[:], c.w[:] = -128, -128
        ctx.matmul_q8(c.args)
        ctx.sync()
        c.verify()
    finally:
        c.free()


@pytest.mark.parametrize("M,N,K", [(1, 22016, 2048), (4, 5120, 8192), (16, 2048, 11008), (37, 17408, 5120),
                                   (130, 4096, 14336), (201, 2560, 2048), (512, 4096, 2048), (1024, 1536, 4096),
                                   (2100, 2304, 1024)])
def test_model_sizes(ctx, ws, M, N, K):
    go(ctx, ws, M, N, K, BF16, lo=-128)


@pytest.mark.parametrize("K", [16, 96, 128, 144, 272, 400, 1104])
@pytest.mark.parametrize("t,N", [(BF16, 4100), (F32, 4103), (F16, 4096)])
def test_more_tiles_than_compute_units(ctx, ws, t, N, K):
    """Tiles of 256 by 256, several a workgroup, the last ones over their neighbours."""
    go(ctx, ws, 4900, N, K, t, bias=t == F16, opad=4, lo=-128)


def test_strides_past_32_bit_offsets(ctx, ws):
    """Rows so far apart that a tile's offsets would not fit 32 bits."""
    M, N, K, far = 130, 70, 272, (1 << 23) + 16
    c = Product(ctx, ws, M, N, K)
    big = ctx.alloc(M * far)
    try:
        for r in range(M):
            big.upload(c.x[r], r * far)
            if r < N:
                big.upload(c.w[r], r * far + 1024)
        c.args.x, c.args.x_stride, c.args.w, c.args.w_stride = big.ptr, far, big.ptr + 1024, far
        ctx.matmul_q8(c.args)
        ctx.sync()
        c.verify()
    finally:
        big.free()
        c.free()


def test_scales_that_are_not_finite(ctx, ws):
    """A row of codes 0 with the scale NaN gives NaN throughout, and no other row."""
    for M in (1, 20, 140):
        c = Product(ctx, ws, M, 150, 128)
        try:
            r = M // 2
            c.x[r] = 0
            c.bufs[0].upload(c.x.reshape(-1))
            c.xs[r] = np.nan
            c.bufs[2].upload(c.xs)
            ctx.matmul_q8(c.args)
            ctx.sync()
            assert np.isnan(c.got()[r]).all()
            c.verify()
        finally:
            c.free()


def test_calls_of_all_sizes_share_a_workspace(ctx, ws):
    """Calls in order, without a wait between them; the counters are 0 again behind them."""
    cases = [Product(ctx, ws, M, N, K, F16, seed=9) for M, N, K in
             [(1, 600, 8192), (130, 520, 4096), (12, 100, 16384), (600, 700, 512), (40, 1000, 8192), (2, 64, 32768)]]
    try:
        for _ in range(3):
            for c in cases:
                ctx.matmul_q8(c.args)
        ctx.sync()
        for c in cases:
            c.verify()
        assert not ws.download(np.int32, 1024).any()
    finally:
        for c in cases:
            c.free()


def test_rows_far_apart(ctx, ws):
    """Rows of x, w and out whose offsets pass 2^32 bytes."""
    M, N, K, far = 3, 3, 256, (3 << 30) + 4096
    c = Product(ctx, ws, M, N, K)
    big = ctx.alloc(2 * far + 8192)
    try:
        for r in range(3):
            big.upload(c.x[r], r * far)
            big.upload(c.w[r], r * far + 1024)
        a = c.args
        a.x, a.x_stride, a.w, a.w_stride = big.ptr, far, big.ptr + 1024, far
        a.out, a.out_stride = big.ptr + 2048, far // 4
        ctx.matmul_q8(a)
        ctx.sync()
        got = np.stack([big.download(np.float32, N, r * far + 2048) for r in range(M)])
        assert np.array_equal(got, c.ref())
    finally:
        big.free()
        c.free()


@pytest.mark.parametrize("M", [33, 47, 64, 100, 150])
@pytest.mark.parametrize("N,K", [(17411, 1040), (22016, 144), (20011, 16), (5121, 17408), (8195, 4112)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_few_rows_of_many_channels(ctx, ws, M, N, K, t):
    """Tiles whose weights come from memory, whole and in parts."""
    go(ctx, ws, M, N, K, t, bias=M % 2 == 1)
