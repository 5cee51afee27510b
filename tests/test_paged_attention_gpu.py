"""mi355x_paged_attention against 64 bits.

Bound of an output value, with A = sum_j w_j |v_j| and S the largest sum
scale |q_d k_jd| of a row: the output's rounding, half a step of the value; the
weights' rounding, half a step of their type times A, or its square for two
planes (f16 planes end at 2^-24 of the largest weight: n such); scores of hd + 8
f32 roundings of S each, which move every weight, and the sum it is divided by,
by as much; and n + 16 f32 roundings of the sums over n keys."""
import ctypes

import numpy as np
import pytest

import mi355x
import paged_ref
from mi355x import BF16, F16, F32
from paged_ref import HALF_STEP, decode, encode, storage

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, ctx, q_lens, kv_lens, hq, hk, hd, t=BF16, out=None, page=16, hnd=False, gap=0, window=0,
                 softcap=0.0, causal=True, spare_rows=0, qpad=0, seed=0, sharp=1.0, max_added=None, cols=None,
                 n_pages=None):
        rng = np.random.default_rng([seed, len(q_lens), hd, sum(q_lens)])
        out = t if out is None else out
        self.__dict__.update(ctx=ctx, hq=hq, hk=hk, hd=hd, t=t, out_t=out, window=window, softcap=softcap,
                             causal=causal, rng=rng)
        self.offsets = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.kv = np.asarray(kv_lens, np.int32)
        self.T = int(self.offsets[-1]) + spare_rows
        need = [-(-max(0, int(k)) // page) for k in kv_lens]
        n_pages = sum(need) + 3 if n_pages is None else n_pages
        self.pool = paged_ref.Pool(ctx, rng, t, n_pages, page, hk, hd, hnd, gap)
        cols = max(need + [1]) if cols is None else cols
        self.table = np.full((len(q_lens), cols), -1, np.int32)
        order, at = rng.permutation(n_pages), 0
        for s, n in enumerate(need):
            n = min(n, cols)
            self.table[s, :n] = order[at:at + n]
            at += n
        self.qs, self.os = hq * hd + qpad, hq * hd + 8
        self.q = decode(encode(sharp * rng.standard_normal((self.T, hq, hd)), t), t)
        self.scale = hd ** -0.5
        self.ws_bytes = ctx.paged_attention_workspace(hq, hk, hd)
        self.bufs = {}
        self.upload()
        self.struct = self.pool.struct()
        self.args = mi355x.PagedAttentionArgs(
            n_rows=self.T, n_seqs=len(q_lens), n_heads=hq,
            max_added=max(q_lens, default=0) if max_added is None else max_added, q=self.bufs["q"].ptr,
            q_stride=self.qs, pool=mi355x.pointer(self.struct), row_offsets=self.bufs["off"].ptr,
            kv_lens=self.bufs["kv"].ptr, block_table=self.bufs["table"].ptr, table_cols=cols,
            table_stride=self.table.shape[1], scale=self.scale, softcap=softcap, window=window,
            causal=int(causal), out=self.bufs["out"].ptr, out_type=out, out_stride=self.os,
            workspace=self.bufs["ws"].ptr, workspace_bytes=self.ws_bytes)

    def upload(self):
        q = encode(np.full((max(self.T, 1), self.qs), 9.0), self.t)
        q[:self.T, :self.hq * self.hd] = encode(self.q.reshape(self.T, -1), self.t)
        d = self.ctx.to_device
        for k, v in dict(q=q, off=self.offsets, kv=self.kv, table=self.table).items():
            if k in self.bufs:
                self.bufs[k].upload(v)
            else:
                self.bufs[k] = d(v)
        if "out" not in self.bufs:
            self.bufs["out"] = d(encode(np.full(max(self.T, 1) * self.os, 7.0), self.out_t))
            self.bufs["ws"] = d(np.zeros(self.ws_bytes, np.uint8))

    def outputs(self):
        o = decode(self.bufs["out"].download(storage(self.out_t), self.T * self.os), self.out_t).reshape(self.T, -1)
        w = self.hq * self.hd
        assert np.all(o[:, w:] == 7.0), "between the rows"
        real = min(self.T, max(0, int(self.offsets[-1])))
        assert np.all(o[real:] == 7.0), "rows behind the last request"
        return o[:real, :w].reshape(real, self.hq, self.hd)

    def reference(self, **over):
        kw = dict(softcap=self.softcap, window=self.window, causal=self.causal)
        kw.update(over)
        return paged_ref.attention(self.q[:int(self.offsets[-1])], self.pool, self.offsets, self.kv, self.table,
                                   self.scale, **kw)

    def verify(self, what=""):
        got = self.outputs()
        ref, mag, size = self.reference()
        n = int(self.kv.max(initial=0))
        w = HALF_STEP[self.t]
        planes = w * w + (n * 2.0 ** -25 if self.t == F16 else 0) if self.out_t == F32 else w
        f32 = 2.0 ** -24 * (2 * (self.hd + 8) * size[..., None] + n + 16)
        bound = HALF_STEP[self.out_t] * np.abs(ref) + (planes + f32) * mag + (2.0 ** -25 if self.out_t == F16 else 0)
        off = np.abs(got - ref)
        assert np.all(off <= bound), (what, float((off / np.maximum(bound, 1e-30)).max()))
        # in the mean far less: roundings are independent, so three of the type's half steps
        # (f32: of the scores' size) bound the norm of the whole difference
        norm = np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-30)
        most = 3 * max(HALF_STEP[self.out_t], 2.0 ** -24 * 8 * size.max(initial=1))
        assert np.linalg.norm(ref) == 0 or norm <= most, (what, norm, most)

    def run(self):
        self.ctx.paged_attention(self.args)
        self.ctx.sync()
        return self

    def free(self):
        for b in self.bufs.values():
            b.free()
        self.pool.free()


def go(ctx, *a, **kw):
    c = Case(ctx, *a, **kw)
    try:
        c.run().verify(kw)
    finally:
        c.free()


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 2), (4, 4), (7, 1), (32, 1)])
def test_one_token(ctx, hq, hk, hd, t, out):
    go(ctx, [1, 1, 1], [1, 33, 300], hq, hk, hd, t, out)


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("hq,hk", [(2, 2), (8, 2), (7, 1)])
def test_chunks(ctx, hq, hk, hd, t, out):
    go(ctx, [37, 1, 150, 5], [37, 200, 333, 64], hq, hk, hd, t, out)


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("hd,hq,hk,softcap", [(64, 8, 1, 0.0), (96, 16, 2, 25.0), (128, 14, 2, 0.0), (256, 8, 1, 0.0)])
def test_many_rows(ctx, hd, hq, hk, softcap, t, out):
    """Enough head rows for workgroups of 256 of them on every CU, and few ones among them."""
    go(ctx, [700] * 6 + [1, 3] + [997] * 5, [700] * 6 + [900, 50] + [1000] * 5, hq, hk, hd, t, out, softcap=softcap)


@pytest.mark.parametrize("t,out", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("hd,hq,hk", [(96, 2, 1), (128, 14, 2), (128, 4, 4), (256, 2, 1)])
@pytest.mark.parametrize("window,causal", [(0, True), (300, True), (0, False)])
def test_long_chunks_alone(ctx, hd, hq, hk, window, causal, t, out):
    """Many rows of one request: workgroups of 256, their keys in parts."""
    q = -(-2050 * hk // hq)
    go(ctx, [q], [q + 1000], hq, hk, hd, t, out, window=window, causal=causal)


@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("q_lens", [[1, 2], [40, 100]])
def test_scales_of_any_sign(ctx, q_lens, scale):
    c = Case(ctx, q_lens, [300, 130], 4, 2, 64, F16, F32)
    try:
        c.scale = c.args.scale = scale
        c.run().verify(scale)
    finally:
        c.free()


@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4097])
def test_every_length(ctx, kv):
    go(ctx, [1], [kv], 4, 2, 64, F16, F32, page=8)


@pytest.mark.parametrize("q", [2, 3, 8, 9, 15, 16, 17, 31, 33, 64, 65, 127, 129, 200])
def test_every_chunk(ctx, q):
    go(ctx, [q, q], [q, q + 77], 4, 2, 64, F16, F16, page=32)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 64, 256, 4096])
@pytest.mark.parametrize("hnd", [False, True])
def test_pages(ctx, page, hnd):
    go(ctx, [1, 40, 3], [500, 70, 130], 8, 2, 64, page=page, hnd=hnd, gap=8)


@pytest.mark.parametrize("window", [1, 2, 16, 50, 64, 100, 1000])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_windows_and_caps(ctx, window, softcap):
    go(ctx, [1, 90, 4, 300], [700, 90, 333, 301], 4, 2, 64, F16, F32, window=window, softcap=softcap, sharp=3.0)


@pytest.mark.parametrize("q_lens,kv", [([1, 2], [300, 130]), ([40, 100], [300, 130])])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [1e-40, 1e-3, 0.5, 40.0, 50.0, 1000.0, 1e9, 3e38])
def test_caps_of_any_size(ctx, cap, hd, q_lens, kv):
    """Scores far below the cap are as exact as without one."""
    go(ctx, q_lens, kv, 4, 2, hd, F16, F32, softcap=cap)


@pytest.mark.parametrize("window", [0, 30])
def test_not_causal(ctx, window):
    go(ctx, [1, 50, 200], [40, 50, 260], 4, 2, 64, window=window, causal=False)


def test_many_requests_of_all_lengths(ctx):
    rng = np.random.default_rng(1)
    q = rng.integers(0, 4, 300)
    go(ctx, list(q), list(q + rng.integers(0, 200, 300)), 4, 1, 64, F16, F16, page=8)


def test_thousands_of_requests(ctx):
    rng = np.random.default_rng(2)
    q = rng.integers(0, 3, 3000)
    go(ctx, list(q), list(q + rng.integers(0, 40, 3000)), 2, 1, 64, BF16, F32, page=4)


def test_one_long_request_among_short_ones(ctx):
    go(ctx, [1] * 9, [5, 3, 20000, 1, 64, 2, 130, 7, 9], 8, 1, 128, F16, F32)


def test_sharp_scores(ctx):
    go(ctx, [1, 60], [900, 300], 4, 2, 128, BF16, F32, sharp=12.0)


def test_rows_that_see_nothing_and_requests_of_no_length(ctx):
    """Lengths of zero, fewer tokens than rows, none at all: zeros; rows behind
    the last request are left."""
    c = Case(ctx, [1, 0, 3, 2, 20, 40], [0, 50, 1, -4, 7, 0], 4, 2, 64, spare_rows=6)
    try:
        got = c.run().outputs()
        c.verify()
        assert np.all(got[0] == 0) and np.all(got[1:3] == 0) and np.any(got[3] != 0)
        assert np.all(got[4:6] == 0) and np.all(got[6:19] == 0) and np.all(got[26:] == 0)
    finally:
        c.free()


@pytest.mark.parametrize("q_lens,kv", [([1, 1], [40, 77]), ([30, 64], [130, 200]), ([6, 200], [90, 200]),
                                       ([130] * 260, [130] * 259 + [150]), ([1100, 1300], [1100, 1400])])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 20])
def test_tokens_not_seen_do_not_reach_a_row(ctx, q_lens, kv, poison, window):
    """Every slot that no row sees is poisoned, and tokens that some rows see:
    the others' outputs stay as they were, bit for bit."""
    c = Case(ctx, q_lens, kv, 4, 2, 96 if q_lens[0] > 1000 else 64, F16, F16, window=window)
    try:
        clean = c.run().outputs()
        c.verify()
        seen = np.zeros(c.pool.k.shape[:2], bool)
        for s, k in enumerate(kv):
            lo = max(0, k - q_lens[s] + 1 - window) if window else 0
            j = np.arange(lo, k)
            seen[c.table[s][j // 16], j % 16] = True
            if window:  # pages that left the window may be gone from the table
                c.table[s, :lo // 16] = [-1, 2 ** 31 - 1][s % 2]
        c.pool.k[~seen], c.pool.v[~seen] = poison, poison
        # the last token of each request: only its last row sees it
        for s, k in enumerate(kv):
            c.pool.k[c.table[s][(k - 1) // 16], (k - 1) % 16] = poison
            c.pool.v[c.table[s][(k - 1) // 16], (k - 1) % 16] = poison
        c.pool.upload()
        c.struct.k, c.struct.v = (b.ptr for b in c.pool.bufs)
        c.upload()
        got = c.run().outputs()
        last = c.offsets[1:] - 1
        rest = np.setdiff1d(np.arange(c.offsets[-1]), last)
        assert np.array_equal(got[rest], clean[rest])
        assert np.all(np.isnan(got[last]))
    finally:
        c.free()


@pytest.mark.parametrize("q", [1, 5, 70])
def test_pages_outside_the_pool_are_not_seen(ctx, q):
    c = Case(ctx, [q, q], [400, 333], 4, 2, 64, F16, F32)
    try:
        c.table[0, 3], c.table[0, 20], c.table[1, 0] = -1, c.pool.n_pages, -2 ** 31
        c.table[1, 7:9] = 2 ** 31 - 1
        c.upload()
        c.run().verify()
    finally:
        c.free()


def test_tokens_behind_the_tables_columns_are_not_seen(ctx):
    go(ctx, [1, 30], [500, 170], 4, 2, 64, F16, F32, cols=9)


@pytest.mark.parametrize("q_lens,max_added", [([1, 1, 1], 0), ([1, 1, 1], 500), ([90, 1, 7], 1), ([90, 1, 7], 0)])
def test_the_hosts_bound_changes_no_meaning(ctx, q_lens, max_added):
    go(ctx, q_lens, [400, 30, 200], 8, 2, 64, F16, F32, max_added=max_added)


@pytest.mark.parametrize("offsets", [[0, 4, 9], [2, 5, 8]])
def test_offsets_past_the_rows(ctx, offsets):
    """Rows that the offsets name past n_rows are not written, and rows before
    the first offset are left."""
    c = Case(ctx, [3, 4], [60, 50], 4, 2, 64, F16, F32)
    try:
        c.offsets = np.asarray(offsets, np.int32)
        c.upload()
        c.run()
        o = c.bufs["out"].download(np.float32, c.T * c.os).reshape(c.T, -1)[:, :256].reshape(c.T, 4, 64)
        assert np.all(o[:offsets[0]] == 7.0)
        full = np.concatenate([c.q, np.zeros((max(0, offsets[-1] - c.T), 4, 64))])
        ref, mag, _ = paged_ref.attention(full, c.pool, c.offsets, c.kv, c.table, c.scale)
        assert np.allclose(o[offsets[0]:], ref[offsets[0]:c.T], rtol=0, atol=1e-4)
    finally:
        c.free()


def test_a_page_used_by_two_requests(ctx):
    c = Case(ctx, [1, 1, 20], [64, 70, 80], 4, 2, 64, F16, F32)
    try:
        c.table[1, :4] = c.table[0, :4]
        c.table[2, :2] = c.table[0, :2]
        c.upload()
        c.run().verify()
    finally:
        c.free()


def test_far_pages(ctx):
    """Offsets past 2^31 values and past 2^32 bytes: a pool of 3 x 2^31 values
    of which three pages are used."""
    c = Case(ctx, [1, 20], [20, 24], 2, 1, 64, F16, F32, n_pages=3)
    big = None
    stride = 2 ** 31
    try:
        big = ctx.alloc(2 * (2 * stride + c.pool.stride) + 2 * 2 ** 16)
        other = ctx.alloc(2 * (2 * stride + c.pool.stride) + 2 * 2 ** 16)
        for dst, src in ((big, c.pool.bufs[0]), (other, c.pool.bufs[1])):
            for p in range(3):
                mi355x.check(ctx.lib.mi355x_memcpy_d2d(ctx.h, dst.ptr + 2 * p * stride, src.ptr + 2 * p * c.pool.stride,
                                                       2 * c.pool.stride))
        c.table[:] = -1
        c.table[0, :2], c.table[1, :2] = [2, 0], [1, 2]
        c.upload()
        c.struct.k, c.struct.v, c.struct.page_stride = big.ptr, other.ptr, stride
        c.run().verify()
        other.free()
    finally:
        if big:
            big.free()
        c.free()


def test_the_same_call_gives_the_same_bits(ctx):
    c = Case(ctx, [1] * 5 + [70, 300], [9000, 3, 800, 77, 1, 900, 301], 8, 2, 128, BF16, F32)
    try:
        a = c.run().outputs()
        for _ in range(3):
            assert np.array_equal(c.run().outputs(), a)
    finally:
        c.free()


def hip_check(rc, what):
    assert rc == 0, f"{what}: hipError_t {rc}"


class Graph:
    """What the context's stream records between enter and exit, replayed on a stream of its own."""

    def __init__(self, ctx):
        self.ctx, self.hip = ctx, ctypes.CDLL("libamdhip64.so")
        self.graph, self.ex, self.stream = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()

    def __enter__(self):
        self.ctx.sync()
        self.own = ctypes.c_void_p(self.ctx.lib.mi355x_ctx_stream(self.ctx.h))
        hip_check(self.hip.hipStreamBeginCapture(self.own, 1), "begin capture")
        return self

    def __exit__(self, *exc):
        hip_check(self.hip.hipStreamEndCapture(self.own, ctypes.byref(self.graph)), "end capture")
        hip_check(self.hip.hipGraphInstantiate(ctypes.byref(self.ex), self.graph, None, None, ctypes.c_size_t(0)),
                  "instantiate")
        hip_check(self.hip.hipStreamCreateWithFlags(ctypes.byref(self.stream), 1), "stream")

    def launch(self):
        hip_check(self.hip.hipGraphLaunch(self.ex, self.stream), "launch")

    def wait(self):
        hip_check(self.hip.hipStreamSynchronize(self.stream), "synchronize")

    def free(self):
        for fn, h in (("hipGraphExecDestroy", self.ex), ("hipGraphDestroy", self.graph),
                      ("hipStreamDestroy", self.stream)):
            if h:
                getattr(self.hip, fn)(h)


def test_replays_take_new_lengths_beside_the_contexts_calls(ctx):
    """A captured call replayed on another stream, with lengths that change
    between replays, while the context runs calls of its own (a workspace each)."""
    c = Case(ctx, [1, 1, 40, 3], [3000, 2, 700, 90], 8, 2, 64, F16, F32)
    d = Case(ctx, [1, 60], [2500, 61], 8, 2, 64, F16, F32, seed=9)
    g = Graph(ctx)
    try:
        own = d.run().outputs()
        with g:
            ctx.paged_attention(c.args)
        for kv in ([3000, 2, 700, 90], [1, 1, 40, 3], [2222, 0, 41, 33], [16, 2, 699, 0]):
            c.kv = np.asarray(kv, np.int32)
            c.upload()
            ctx.sync()
            g.launch()
            for _ in range(3):
                ctx.paged_attention(d.args)
            g.wait()
            ctx.sync()
            c.verify(kv)
            assert np.array_equal(d.outputs(), own)
    finally:
        g.free()
        c.free()
        d.free()


def test_two_contexts_at_once(ctx):
    with mi355x.Context(0) as other:
        c = Case(ctx, [1, 90], [5000, 300], 8, 2, 64, F16, F32)
        d = Case(other, [1, 80], [4000, 200], 8, 2, 64, F16, F32, seed=3)
        try:
            for _ in range(4):
                ctx.paged_attention(c.args)
                other.paged_attention(d.args)
            ctx.sync()
            other.sync()
            c.verify()
            d.verify()
        finally:
            c.free()
            d.free()
