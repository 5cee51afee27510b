"""Attention of single tokens on long contexts, where workgroups get more than one unit
of 128 keys on purpose and rows are cut at the beginning of a workgroup's stretch and
behind it: against 64 bits, with the sharing out worked out here to see that the cases
are such ones."""
import math

import numpy as np
import pytest

from mi355x import BF16, F16, F32
from test_paged_attention_gpu import Case

pytestmark = pytest.mark.gpu

UNIT, THREADS, ROWS = 128, 256, 16  # keys of a unit, a workgroup's threads, its head rows


def shared_out(kv, hq, hk, hd, window, q=1):
    """(units of a workgroup wanted, whether a row is cut that begins a stretch, whether one
    is that begins behind a stretch's beginning)."""
    group = hq // hk
    assert q * group <= ROWS
    # per request and KV head: units from the first key that its first row sees
    tiles = [-(-(n - max(0, n - q - window + 1 if window else 0)) // UNIT) for n in kv for _ in range(hk)]
    teams = max(1, THREADS // (min(ROWS, q * group) * (hd // 4)))
    total = sum(tiles)
    wanted = math.sqrt(total / (12 * teams * len(kv) * hk)) + 0.5
    # fewer workgroups than the smallest number that runs at once on 256 CUs, or their number would count
    groups = -(-total // int(wanted))
    assert groups <= 256
    each, longer = divmod(total, groups)
    starts = [each * g + min(g, longer) for g in range(groups + 1)]
    at, begins, behind = 0, False, False
    for n in tiles:
        g = max(i for i in range(groups) if starts[i] <= at)
        if at + n > starts[g + 1]:  # cut
            begins |= at == starts[g]
            behind |= at != starts[g]
        at += n
    return wanted, begins, behind


@pytest.mark.parametrize("t,out", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("kv,hq,hk,window", [
    ([16000], 16, 1, 0), ([40000], 16, 1, 0), ([20011], 16, 1, 15000), ([5000, 4100, 6001, 4700], 32, 2, 0),
    ([9000, 4100, 12000], 48, 3, 7000), ([5003, 9000, 4999, 7001, 6000], 16, 1, 0)])
def test_stretches_of_several_units(ctx, kv, hq, hk, window, hd, t, out):
    wanted, begins, behind = shared_out(kv, hq, hk, hd, window)
    assert wanted >= 2 and begins and (behind or len(kv) * hk == 1)
    c = Case(ctx, [1] * len(kv), kv, hq, hk, hd, t, out, page=64, window=window)
    try:
        c.run().verify()
    finally:
        c.free()


@pytest.mark.parametrize("hd", [64, 256])
def test_a_few_tokens_on_long_contexts(ctx, hd):
    kv = [7000, 11000, 6500]
    wanted, begins, behind = shared_out(kv, 4, 1, hd, 0, 4)
    assert wanted >= 2 and begins and behind
    c = Case(ctx, [4] * 3, kv, 4, 1, hd, F16, F32, page=64)
    try:
        c.run().verify()
    finally:
        c.free()
