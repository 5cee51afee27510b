"""The operators of mi355x-layer.h one behind the other, as a layer and a model's
end use them: an attention's output in 8 bits, its projection, the residual's
addition with the norm, gate and up, the gated row, down, the last norm, the
vocabulary, and log probabilities.

Every step up to the logits has stated roundings, so that numpy's logits are the
same bits; the bounds of the log probabilities are those of test_logprobs_gpu.py."""
import ctypes

import numpy as np
import pytest

import layer_ref
import mi355x
from layer_ref import decode, encode, storage
from mi355x import BF16, F32
from test_logprobs_gpu import Logits
from test_paged_attention_gpu import Graph

pytestmark = pytest.mark.gpu
H, F, V, TOP = 512, 1376, 4003, 9
EPS = 1e-5


class Weights:
    def __init__(self, ctx, seed):
        rng = np.random.default_rng(seed)
        self.ctx, self.bufs = ctx, []
        mat = lambda n, k: (rng.integers(-127, 128, (n, k)).astype(np.int8),  # noqa: E731
                            (np.exp(0.2 * rng.standard_normal(n)) * 0.02 / 127 * np.sqrt(512 / k)).astype(np.float32))
        self.o, self.gate_up, self.down, self.vocab = mat(H, H), mat(2 * F, H), mat(H, F), mat(V, H)
        self.bias = rng.standard_normal(2 * F).astype(np.float32) * np.float32(0.1)
        self.norms = [(1 + 0.2 * rng.standard_normal(H)).astype(np.float32) for _ in range(2)]
        self.dev = {n: [self.put(a) for a in getattr(self, n)] for n in ("o", "gate_up", "down", "vocab", "norms")}
        self.dev_bias = self.put(self.bias)

    def put(self, a):
        self.bufs.append(self.ctx.to_device(a))
        return self.bufs[-1].ptr

    def free(self):
        for b in self.bufs:
            b.free()


class Run:
    """The buffers of a run of T rows on a context, its calls, and numpy's results for the same inputs."""

    def __init__(self, ctx, w, T):
        self.ctx, self.w, self.T, self.bufs = ctx, w, T, []
        self.att, self.res = self.alloc(T * H, BF16), self.alloc(T * H, F32)
        self.tok = self.alloc(T, F32)
        self.code = [self.alloc(T * n, None) for n in (H, H, F, H)]
        self.scale = [self.alloc(T, F32) for _ in range(4)]
        self.proj, self.gu, self.down = self.alloc(T * H, BF16), self.alloc(T * 2 * F, BF16), self.alloc(T * H, BF16)
        self.logits = self.alloc(T * V, F32)
        self.lp, self.ent = self.alloc(T, F32), self.alloc(T, F32)
        self.top, self.top_lp = self.alloc(T * TOP, F32), self.alloc(T * TOP, F32)
        self.ws, self.lws = self.zeroed(ctx.matmul_q8_workspace()), self.zeroed(ctx.logprobs_workspace())

    def alloc(self, n, t):
        b = self.ctx.alloc(n * (1 if t is None else np.dtype(storage(t)).itemsize))
        self.bufs.append(b)
        return b

    def zeroed(self, n):
        b = self.alloc(n, None)
        mi355x.check(self.ctx.lib.mi355x_fill(self.ctx.h, b.ptr, 0, n))
        return b

    def inputs(self, seed):
        rng = np.random.default_rng([seed, self.T])
        self.a = encode(rng.standard_normal((self.T, H)), BF16)
        self.r = (3 * rng.standard_normal((self.T, H))).astype(np.float32)
        self.tokens = rng.integers(0, V, self.T).astype(np.int32)
        self.att.upload(self.a)
        self.res.upload(self.r)
        self.tok.upload(self.tokens)
        return self

    def norm(self, x, t, i, residual, norm):
        self.ctx.norm_q8(mi355x.NormQ8Args(
            n_rows=self.T, n=H, type=t, x=x.ptr, x_stride=H, residual_type=F32, residual=self.res.ptr if residual else None,
            residual_stride=H, residual_out=self.res.ptr if residual else None, residual_out_stride=H, eps=EPS, norm=norm,
            q=self.code[i].ptr, q_stride=H, scales=self.scale[i].ptr))

    def matmul(self, i, k, name, n, out, t, bias=None):
        w, ws = self.w.dev[name]
        self.ctx.matmul_q8(mi355x.MatmulQ8Args(
            n_rows=self.T, n_out=n, k=k, x=self.code[i].ptr, x_stride=k, x_scales=self.scale[i].ptr, w=w, w_stride=k,
            w_scales=ws, bias=bias, out=out.ptr, out_type=t, out_stride=n, workspace=self.ws.ptr,
            workspace_bytes=self.ws.nbytes))

    def call(self):
        T, w = self.T, self.w
        self.norm(self.att, BF16, 0, False, None)
        self.matmul(0, H, "o", H, self.proj, BF16)
        self.norm(self.proj, BF16, 1, True, w.dev["norms"][0])
        self.matmul(1, H, "gate_up", 2 * F, self.gu, BF16, w.dev_bias)
        self.ctx.swiglu_q8(mi355x.SwigluQ8Args(n_rows=T, n=F, type=BF16, gate=self.gu.ptr, gate_stride=2 * F,
                                               up=self.gu.ptr + 2 * F, up_stride=2 * F, q=self.code[2].ptr, q_stride=F,
                                               scales=self.scale[2].ptr))
        self.matmul(2, F, "down", H, self.down, BF16)
        self.norm(self.down, BF16, 3, True, w.dev["norms"][1])
        self.matmul(3, H, "vocab", V, self.logits, F32)
        self.ctx.logprobs(mi355x.LogprobsArgs(
            n_rows=T, n_vocab=V, type=F32, logits=self.logits.ptr, stride=V, scale=1.0, n_tokens=1, tokens=self.tok.ptr,
            token_logprobs=self.lp.ptr, entropy=self.ent.ptr, n_top=TOP, top_tokens=self.top.ptr,
            top_logprobs=self.top_lp.ptr, workspace=self.lws.ptr, workspace_bytes=self.lws.nbytes))

    def expected(self):
        def quantized(t, factor=1.0):
            c, s, _ = layer_ref.codes_of(t)
            return c, (s * factor).astype(np.float32)

        def normed(x, residual, norm):
            h, t, factor = layer_ref.norm_rows(decode(x, BF16), residual, F32, norm, EPS)
            return (h.astype(np.float32), *quantized(t, factor))

        w = self.w
        y = layer_ref.matmul(*self.mixed(quantized(decode(self.a, BF16)), w.o), None, BF16)
        h, c, s = normed(y, self.r, w.norms[0])
        gu = decode(layer_ref.matmul(*self.mixed((c, s), w.gate_up), w.bias, BF16), BF16)
        y = layer_ref.matmul(*self.mixed(quantized(layer_ref.swiglu(gu[:, :F], gu[:, F:])), w.down), None, BF16)
        h, c, s = normed(y, h, w.norms[1])
        return h, layer_ref.matmul(*self.mixed((c, s), w.vocab), None, F32)

    @staticmethod
    def mixed(x, w):
        return x[0], w[0], x[1], w[1]

    def verify(self, ctx):
        h, logits = self.expected()
        assert np.array_equal(self.res.download(np.float32, self.T * H).reshape(self.T, H), h)
        assert np.array_equal(self.logits.download(np.float32, self.T * V).reshape(self.T, V), logits)
        # the same logits through one call whose outputs are checked
        c = Logits(ctx, self.lws, logits, F32, top=TOP, tokens=self.tokens[:, None])
        try:
            ctx.logprobs(c.args)
            ctx.sync()
            c.verify()
            for mine, other, t, n in ((self.lp, c.lp, np.float32, 1), (self.ent, c.ent, np.float32, 1),
                                      (self.top, c.tt, np.int32, TOP), (self.top_lp, c.tlp, np.float32, TOP)):
                assert np.array_equal(mine.download(t, self.T * n), other.download(t, self.T * n))
        finally:
            c.free()
        assert not self.ws.download(np.int32, 1024).any() and not self.lws.download(np.int32, 1024).any()

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.fixture(scope="module")
def weights(ctx):
    w = Weights(ctx, 3)
    yield w
    w.free()


@pytest.mark.parametrize("T", [1, 2, 16, 37, 64, 130, 300])
def test_a_layer_and_the_models_end(ctx, weights, T):
    r = Run(ctx, weights, T)
    try:
        for seed in (1, 2):
            r.inputs(seed)
            r.call()
            ctx.sync()
            r.verify(ctx)
    finally:
        r.free()


@pytest.mark.parametrize("T", [1, 40, 140])
def test_replays_beside_the_contexts_calls(ctx, weights, T):
    """The run captured into a graph and replayed on another stream with new inputs, while the context has a
    run of its own (workspaces of their own): every replay is the eager run's bits."""
    r, own = Run(ctx, weights, T), Run(ctx, weights, T + 3)
    g = Graph(ctx)
    try:
        own.inputs(50)
        with g:
            r.call()
        for seed in range(4):
            r.inputs(seed)
            own.res.upload(own.r)
            ctx.sync()
            g.launch()
            own.call()
            g.wait()
            ctx.sync()
            r.verify(ctx)
            own.verify(ctx)
    finally:
        g.free()
        r.free()
        own.free()


def test_two_contexts_at_once(ctx, weights):
    with mi355x.Context(0) as other:
        a, b = Run(ctx, weights, 70), Run(other, weights, 1)
        try:
            for seed in range(3):
                a.inputs(seed)
                b.inputs(seed + 10)
                ctx.sync()
                other.sync()
                a.call()
                b.call()
                ctx.sync()
                other.sync()
                a.verify(ctx)
                b.verify(ctx)
        finally:
            a.free()
            b.free()


@pytest.mark.parametrize("entry", ["mi355x_norm_q8", "mi355x_swiglu_q8", "mi355x_matmul_q8", "mi355x_logprobs"])
def test_an_injected_fault_is_reported(ctx, weights, entry):
    """The call fails before any device work, and the next one runs."""
    r = Run(ctx, weights, 2)
    try:
        r.inputs(7)
        mi355x.inject_fault(entry, mi355x.HIP_ERROR_LAUNCH_FAILURE)
        with pytest.raises(mi355x.Mi355xError):
            r.call()
        assert "[injected]" in mi355x.last_error()
        r.inputs(8)
        r.call()
        ctx.sync()
        r.verify(ctx)
    finally:
        r.free()
