"""mi355x_kv_plan against a row-by-row numpy form: all whole numbers, equal."""
import numpy as np
import pytest

import mi355x
import paged_ref

pytestmark = pytest.mark.gpu


class Plan:
    def __init__(self, ctx, cached, added, page, cols, n_rows, free, head, table, stride=None, in_place=False):
        n = len(cached)
        self.ctx, self.n, self.cols, self.n_rows, self.stride = ctx, n, cols, n_rows, stride or cols
        wide = np.full((max(n, 1), max(self.stride, 1)), -7, np.int32)
        wide[:n, :cols] = table
        i32 = lambda v: ctx.to_device(np.asarray(v, np.int32))  # noqa: E731
        b = dict(cached=i32(cached), added=i32(added), block_table=i32(wide), free_pages=i32(free),
                 free_head=i32([head]), row_offsets=i32(np.full(n + 1, -9)), positions=i32(np.full(n_rows + 1, -9)),
                 slots=ctx.to_device(np.full(n_rows + 1, -9, np.int64)), status=i32([-9]))
        b["kv_lens"] = b["cached"] if in_place else i32(np.full(max(n, 1), -9))
        b["free_head_out"] = b["free_head"] if in_place else i32([-9])
        self.b = b
        self.args = mi355x.KvPlanArgs(n_seqs=n, page_tokens=page, table_cols=cols, n_free=len(free),
                                      table_stride=self.stride, n_rows=n_rows, **{k: v.ptr for k, v in b.items()})

    def run(self):
        self.ctx.kv_plan(self.args)
        self.ctx.sync()
        return self.outputs()

    def outputs(self):
        g = lambda k, c, t=np.int32: self.b[k].download(t, c)  # noqa: E731
        wide = g("block_table", max(self.n, 1) * max(self.stride, 1)).reshape(max(self.n, 1), -1)
        assert np.all(wide[:, self.cols:] == -7), "behind the table's columns"
        pos, slots = g("positions", self.n_rows + 1), g("slots", self.n_rows + 1, np.int64)
        assert pos[-1] == -9 and slots[-1] == -9, "behind the rows"
        return dict(row_offsets=g("row_offsets", self.n + 1), kv_lens=g("kv_lens", self.n),
                    table=wide[:self.n, :self.cols], head=int(g("free_head_out", 1)[0]), positions=pos[:-1],
                    slots=slots[:-1], status=int(g("status", 1)[0]))

    def free(self):
        for b in {id(v): v for v in self.b.values()}.values():
            b.free()


def lengths(rng, n, cached_hi, added_hi):
    return rng.integers(0, cached_hi + 1, n), rng.integers(0, added_hi + 1, n)


def inputs(rng, cached, added, page, spare_cols=1):
    """A table that holds the cached tokens' pages, and a free list with used entries."""
    held = -(-cached // page)
    need = -(-(cached + added) // page)
    cols = int(max(need.max(initial=0), 1)) + spare_cols
    pages = rng.permutation(int(held.sum() + (need - held).sum()) + 9).astype(np.int32)
    table = np.full((len(cached), cols), -1, np.int32)
    table[np.arange(cols) < held[:, None]] = pages[:held.sum()]
    free = np.concatenate([np.full(5, 10 ** 6, np.int32), pages[held.sum():]])
    return table, free, 5


def equal(got, ref):
    assert got["status"] == 0
    for k, v in ref.items():
        assert np.array_equal(got[k], v), k


@pytest.mark.parametrize("n,cached_hi,added_hi,page,pad", [
    (1, 0, 1, 16, 0), (1, 100, 1, 1, 0), (3, 0, 70, 8, 5), (64, 900, 1, 16, 0), (65, 50, 9, 64, 1),
    (257, 300, 40, 32, 3), (1024, 40, 3, 8, 0), (1025, 40, 3, 8, 2), (2500, 33, 5, 4, 700), (7, 3000, 4000, 256, 11),
    (40, 0, 0, 16, 6), (2, 5, 90000, 1, 4), (1100, 9, 300, 2, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ctx, n, cached_hi, added_hi, page, pad, in_place):
    rng = np.random.default_rng([n, page])
    cached, added = lengths(rng, n, cached_hi, added_hi)
    if n == 1:
        added[:] = 1
    table, free, head = inputs(rng, cached, added, page)
    n_rows = int(added.sum()) + pad
    ref = paged_ref.plan(cached, added, page, table, free, head, n_rows)
    p = Plan(ctx, cached, added, page, table.shape[1], n_rows, free, head, table, table.shape[1] + 3, in_place)
    try:
        equal(p.run(), ref)
    finally:
        p.free()


def test_no_requests_and_no_rows(ctx):
    p = Plan(ctx, [], [], 16, 0, 5, [1], 1, np.zeros((0, 0), np.int32))
    try:
        got = p.run()
        assert got["status"] == 0 and got["head"] == 1 and list(got["row_offsets"]) == [0]
        assert np.all(got["positions"] == 0) and np.all(got["slots"] == -1)
    finally:
        p.free()


@pytest.mark.parametrize("n", [3, 1500])
@pytest.mark.parametrize("what,bits", [
    ("negative", mi355x.KV_BAD_LENGTH), ("past 2^31", mi355x.KV_BAD_LENGTH), ("rows", mi355x.KV_ROWS),
    ("columns", mi355x.KV_TABLE), ("pages", mi355x.KV_PAGES), ("head", mi355x.KV_PAGES), ("low head", mi355x.KV_PAGES),
    ("two", mi355x.KV_ROWS | mi355x.KV_PAGES)])
def test_what_does_not_fit_takes_nothing(ctx, n, what, bits):
    rng = np.random.default_rng(n)
    cached, added = rng.integers(1, 50, n), rng.integers(1, 9, n)
    table, free, head = inputs(rng, cached, added, 8, 0)
    rows, cols = int(added.sum()), table.shape[1]
    if what == "negative":
        added[n // 2] = -1
    elif what == "past 2^31":
        cached[n - 1] = 2 ** 31 - 1
    elif what == "columns":
        cols -= 1
    elif what == "head":
        head = len(free) + 1
    elif what == "low head":
        head = -1
    if what in ("rows", "two"):
        rows -= 1
    if what in ("pages", "two"):
        need = int((-(-(cached + added) // 8) - -(-cached // 8)).sum())
        free = free[:head + need - 1]
    p = Plan(ctx, cached, added, 8, cols, rows, free, head, table[:, :cols], cols + 1)
    try:
        got = p.run()
        assert got["status"] == bits
        assert got["head"] == head and np.all(got["row_offsets"] == 0) and np.array_equal(got["table"], table[:, :cols])
        assert np.array_equal(got["kv_lens"], np.maximum(cached, 0))
        assert np.all(got["slots"] == -1) and np.all(got["positions"] == 0)
    finally:
        p.free()


def test_steps_in_place_walk_through_the_pages(ctx):
    """A decode loop: every step in place adds a token or a few to each request."""
    rng = np.random.default_rng(5)
    n, page, steps = 9, 4, 12
    cached = np.zeros(n, np.int64)
    added = rng.integers(0, 4, n)
    table, free = np.full((n, 16), -1, np.int32), rng.permutation(400).astype(np.int32)
    head = 0
    p = Plan(ctx, cached, added, page, 16, int(added.sum()) + 2, free, head, table, 16, True)
    try:
        for _ in range(steps):
            ref = paged_ref.plan(cached, added, page, table, free, head, p.n_rows)
            equal(p.run(), ref)
            cached, table, head = ref["kv_lens"].astype(np.int64), ref["table"], ref["head"]
    finally:
        p.free()
