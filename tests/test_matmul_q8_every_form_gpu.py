"""mi355x_matmul_q8 in each of its kernel forms, whole and in parts of k: the sizes
of matmul_q8_sizes.py, which the CPU tests hold to the forms that they are named
for.  Every bit is the stated one."""
import numpy as np
import pytest

from matmul_q8_sizes import SIZES
from mi355x import BF16, F16, F32
from test_matmul_q8_gpu import Product, ws  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
COUNTERS = 32 * 1024  # ints at the workspace's begin: a counter of 32 ints for each of 1024 tiles
LARGE = SIZES["256x256"]
OTHERS = [(form, *size) for form, sizes in SIZES.items() if form != "256x256" for size in sizes]


def go(ctx, ws, *a, calls=1, **kw):  # noqa: F811
    c = Product(ctx, ws, *a, **kw)
    try:
        for _ in range(calls):
            ctx.matmul_q8(c.args)
        ctx.sync()
        c.verify()
        assert not ws.download(np.int32, COUNTERS).any()
    finally:
        c.free()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", LARGE)
def test_large_tiles(ctx, ws, M, N, K, t):  # noqa: F811
    """One tile a workgroup and several, their prefetch under the outputs' stores, the last
    ones over their neighbours, and a k that ends inside a stage."""
    go(ctx, ws, M, N, K, t, bias=t != BF16, lo=-128)


@pytest.mark.parametrize("M,N,K", [(777, 30001, 272), (513, 40009, 384)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_large_tiles_of_rows_apart(ctx, ws, M, N, K, t):  # noqa: F811
    go(ctx, ws, M, N, K, t, bias=t == BF16, xpad=16, wpad=112, opad=5, oshift=1)


@pytest.mark.parametrize("form,M,N,K", OTHERS)
@pytest.mark.parametrize("t", [F32, BF16])
def test_other_forms(ctx, ws, form, M, N, K, t):  # noqa: F811
    """Calls one behind the other find the counters at 0."""
    go(ctx, ws, M, N, K, t, bias=t == F32, opad=3, lo=-128, calls=3)


@pytest.mark.parametrize("form,M,N,K", [o for o in OTHERS if " in " in o[0]])
def test_parts_of_rows_apart(ctx, ws, form, M, N, K):  # noqa: F811
    go(ctx, ws, M, N, K, F16, bias=True, xpad=48, wpad=16, opad=8, oshift=8)
