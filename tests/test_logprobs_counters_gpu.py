"""mi355x_logprobs: every row's counter is 0 again behind calls of many rows in
parts, and of fewer."""
import numpy as np
import pytest

from mi355x import BF16, F32
from test_logprobs_gpu import Logits, logits, ws  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
COUNTERS = 32 * 512  # ints at the workspace's begin: a counter of 32 ints for each of 512 rows


@pytest.mark.parametrize("t,rows", [(F32, (40, 384, 383, 7)), (BF16, (512, 100, 511, 1))])
def test_counters_of_all_rows(ctx, ws, t, rows):  # noqa: F811
    """(384 rows of 32-bit logits and 512 of 16 bits: the most that are cut into parts.)"""
    cases = [Logits(ctx, ws, logits(T, V, 11), t, top=top) for T, V, top in zip(rows, (30000, 9001, 8200, 60000), (5, 0, 20, 64))]
    try:
        for _ in range(3):
            for c in cases:
                ctx.logprobs(c.args)
        ctx.sync()
        for c in cases:
            c.verify()
        a = ws.download(np.int32, COUNTERS + 4096)
        assert not a[:COUNTERS].any() and a[COUNTERS:].any()
    finally:
        for c in cases:
            c.free()
