"""mi355x_norm_q8 where every second quotient is a tie: products h * norm of up to
254 in magnitude have codes of half themselves, to the even one, whatever the
row's root rounds to."""
import numpy as np
import pytest

import mi355x
from layer_ref import HALF_STEP
from mi355x import BF16, F16, F32
from test_row_q8_gpu import Codes, Rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,T", [(5, 3), (64, 300), (2050, 1030), (16391, 5), (40001, 3)])
def test_ties_do_not_see_the_root(ctx, t, n, T):
    rng = np.random.default_rng([n, T])
    w = 2.0 ** rng.integers(-2, 3, n)
    p = rng.integers(-253, 254, (T, n)).astype(np.float64)
    p[:, rng.integers(0, n)] = 254  # 127 * p / 254; at most 8 bits: exact in every type
    x = Rows(ctx, p / w, t, pad=3)
    assert np.array_equal(x.values * w, p)
    c, norm = Codes(ctx, T, n, pad=1), ctx.to_device(w.astype(np.float32))
    try:
        for eps in (0.0, 1e-6, 0.3):
            ctx.norm_q8(mi355x.NormQ8Args(n_rows=T, n=n, type=t, x=x.ptr, x_stride=x.stride, eps=eps, norm=norm.ptr,
                                          q=c.ptr, q_stride=c.stride, scales=c.s.ptr))
            ctx.sync()
            q, s = c.get()
            assert np.array_equal(q, np.rint(p / 2).astype(np.int8))
            root = np.sqrt((x.values ** 2).mean(1) + np.float64(np.float32(eps)))
            # a step of f32 and the 64-bit sum, root and quotients
            assert np.all(np.abs(s - 2 / root) <= (HALF_STEP[F32] + 1e-12) * (2 / root))
    finally:
        x.buf.free()
        c.free()
        norm.free()
