"""The run of test_layer_run_gpu.py at sizes where the down product's k and the
logits' rows are cut into parts, which meet in the workspaces: eager, replayed
from a graph beside the context's own calls, and on two contexts at once."""
import numpy as np
import pytest

import mi355x
import test_layer_run_gpu as layer
from test_layer_run_gpu import Run, Weights
from test_paged_attention_gpu import Graph

pytestmark = pytest.mark.gpu
MATMUL_COUNTERS, LOGPROBS_COUNTERS = 32 * 1024, 32 * 512  # ints at a workspace's begin


@pytest.fixture(scope="module")
def weights(ctx):
    with pytest.MonkeyPatch.context() as p:
        p.setattr(layer, "F", 4224)
        p.setattr(layer, "V", 20011)
        w = Weights(ctx, 4)
        yield w
        w.free()


def check(ctx, r):
    """The run's results, and that both workspaces were used and left with their counters at 0."""
    r.verify(ctx)
    for ws, counters in ((r.ws, MATMUL_COUNTERS), (r.lws, LOGPROBS_COUNTERS)):
        a = ws.download(np.int32, counters + 4096)
        assert not a[:counters].any() and a[counters:].any()


@pytest.mark.parametrize("T", [37, 64, 140, 300])
def test_a_layer_and_the_models_end_in_parts(ctx, weights, T):
    r = Run(ctx, weights, T)
    try:
        for seed in (1, 2):
            r.inputs(seed)
            r.call()
            ctx.sync()
            check(ctx, r)
    finally:
        r.free()


@pytest.mark.parametrize("T", [37, 140])
def test_replays_beside_the_contexts_calls_in_parts(ctx, weights, T):
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
            check(ctx, r)
            check(ctx, own)
    finally:
        g.free()
        r.free()
        own.free()


def test_two_contexts_at_once_in_parts(ctx, weights):
    with mi355x.Context(0) as other:
        a, b = Run(ctx, weights, 70), Run(other, weights, 33)
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
                check(ctx, a)
                check(other, b)
        finally:
            a.free()
            b.free()
