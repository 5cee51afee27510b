"""The kernels' index arithmetic (csrc/paged_index.h), compiled for the CPU: no
row, token, page or slot outside its buffer, whatever the lengths and tables."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xdna.cpp_amd", "csrc")
SRC = r"""
#include "paged_index.h"
using namespace mi355x;
extern "C" {
int c_seq_of_row(const int32_t *o, int n, int64_t r) { return seq_of_row(o, n, r); }
void c_seq_rows(int64_t b, int64_t e, int64_t t, int64_t *out) {
    SeqRows s = seq_rows(b, e, t);
    out[0] = s.first, out[1] = s.n, out[2] = s.lo, out[3] = s.hi;
}
void c_visible(int64_t p, int64_t kv, int64_t reach, int w, int causal, int64_t *out) {
    KeyRange r = visible_keys(p, kv, reach, w, causal != 0);
    out[0] = r.lo, out[1] = r.hi;
}
int c_page(int32_t p, int64_t n) { return page_in_pool(p, n); }
int c_slot(int64_t s, int64_t n, int shift) { return slot_in_pool(s, n, shift); }
int32_t c_divided(int32_t n, uint32_t d) { return divided(n, fast_div(d)); }
int64_t c_stretch(int64_t total, int groups, int64_t g) { return stretch_begin(stretches(total, groups), g); }
int64_t c_stretch_of(int64_t total, int groups, int64_t u) { return stretch_of(stretches(total, groups), u); }
int64_t c_pages(int64_t n, int shift) { return pages_of(n, shift); }
}
"""


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    d = tmp_path_factory.mktemp("idx")
    (d / "idx.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    f"-I{CSRC}", str(d / "idx.cpp"), "-o", str(d / "idx.so")], check=True)
    lib = ctypes.CDLL(str(d / "idx.so"))
    i64 = ctypes.c_int64
    lib.c_seq_of_row.argtypes = [ctypes.c_void_p, ctypes.c_int, i64]
    lib.c_seq_rows.argtypes = [i64, i64, i64, ctypes.c_void_p]
    lib.c_visible.argtypes = [i64, i64, i64, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    lib.c_page.argtypes = [ctypes.c_int32, i64]
    lib.c_slot.argtypes = [i64, i64, ctypes.c_int]
    lib.c_divided.argtypes = [ctypes.c_int32, ctypes.c_uint32]
    for f in (lib.c_stretch, lib.c_stretch_of):
        f.argtypes, f.restype = [i64, ctypes.c_int, i64], i64
    lib.c_pages.argtypes, lib.c_pages.restype = [i64, ctypes.c_int], i64
    return lib


def test_row_to_request(idx):
    rng = np.random.default_rng(0)
    for n in (1, 2, 3, 17, 100):
        lens = rng.integers(0, 4, n)
        off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        owner = np.repeat(np.arange(n), lens)
        for r in range(-2, int(off[-1]) + 3):
            want = owner[r] if 0 <= r < off[-1] else -1
            assert idx.c_seq_of_row(off.ctypes.data, n, r) == want
    # offsets that do not ascend: any answer names an existing request
    for _ in range(200):
        off = rng.integers(-2 ** 31, 2 ** 31, 9).astype(np.int32)
        assert -1 <= idx.c_seq_of_row(off.ctypes.data, 8, int(rng.integers(-5, 2 ** 31))) < 8
    assert idx.c_seq_of_row(None, 0, 0) == -1


def test_rows_stay_inside(idx):
    out = np.zeros(4, np.int64)
    ends = [-2 ** 31, -5, -1, 0, 1, 7, 8, 9, 2 ** 31 - 1]
    for b in ends:
        for e in ends:
            for t in (0, 1, 8, 2 ** 31 - 1):
                idx.c_seq_rows(b, e, t, out.ctypes.data)
                first, n, lo, hi = out
                assert n == max(0, e - b) and 0 <= lo <= hi <= n
                if hi > lo:
                    assert 0 <= first + lo and first + hi <= t
                # every row inside is covered
                assert hi - lo == max(0, min(e, t) - max(b, 0)) if e > b else hi == lo


def test_visible_tokens(idx):
    out = np.zeros(2, np.int64)
    for pos in (-7, -1, 0, 1, 5, 9, 2 ** 31 - 2):
        for kv in (-3, 0, 1, 6, 10, 2 ** 31 - 1):
            for reach in (0, 4, 8, 2 ** 31 - 1):
                for w in (0, 1, 3, 2 ** 31 - 1):
                    for causal in (0, 1):
                        idx.c_visible(pos, kv, reach, w, causal, out.ctypes.data)
                        lo, hi = out
                        assert 0 <= lo <= hi <= min(max(kv, 0), reach)
                        for j in (0, 1, 3, 4, 5, 6, 7, 9, 10, 2 ** 31 - 2):
                            see = j < kv and j < reach and (not causal or j <= pos) and (not w or j > pos - w)
                            assert (lo <= j < hi) == see, (pos, kv, reach, w, causal, j)


def test_pages_and_slots(idx):
    for n in (0, 1, 5, 2 ** 31 - 1):
        for p in (-2 ** 31, -1, 0, 1, 4, 5, 2 ** 31 - 1):
            assert bool(idx.c_page(p, n)) == (0 <= p < n)
        for shift in (0, 4, 16):
            for s in (-2 ** 63, -1, 0, n << shift, (n << shift) - 1, (n << shift) + 1, 2 ** 63 - 1):
                assert bool(idx.c_slot(s, n, shift)) == (0 <= s < n << shift)
    assert [idx.c_pages(n, 4) for n in (0, 1, 16, 17, 2 ** 31 - 1)] == [0, 1, 1, 2, 2 ** 27]


def test_division_by_a_product(idx):
    rng = np.random.default_rng(2)
    most = 2 ** 31 - 1
    for d in [1, 2, 3, 5, 6, 7, 8, 9, 12, 127, 128, 641, 65535, 65536, *map(int, rng.integers(1, 65537, 50))]:
        ns = {0, 1, d - 1, d, d + 1, most, most - 1, most // d * d, most // d * d - 1, *map(int, rng.integers(0, most, 60))}
        for n in ns:
            assert idx.c_divided(n, d) == n // d, (n, d)


@pytest.mark.parametrize("groups", [1, 2, 5, 768])
def test_stretches_cover_the_line(idx, groups):
    for total in (0, 1, 4, 767, 768, 769, 10 ** 6 + 7, 2 ** 33 + 5):
        at = [idx.c_stretch(total, groups, g) for g in range(groups + 1)]
        assert at[0] == 0 and at[-1] == total
        size = np.diff(at)
        assert size.min() >= 0 and size.max() - size.min() <= 1 and (np.diff(size) <= 0).all()
        for g in range(0, groups, max(1, groups // 9)):
            for u in {at[g], at[g + 1] - 1} if at[g + 1] > at[g] else ():
                assert idx.c_stretch_of(total, groups, u) == g
