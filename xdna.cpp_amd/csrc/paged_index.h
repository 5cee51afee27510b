// Index arithmetic of the paged KV cache, shared by the kernels and by the CPU
// tests (no HIP in here but the function attributes).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define MI355X_HD __host__ __device__ __forceinline__
#else
#define MI355X_HD inline
#endif

namespace mi355x {

MI355X_HD int64_t idx_min(int64_t a, int64_t b) { return a < b ? a : b; }
MI355X_HD int64_t idx_max(int64_t a, int64_t b) { return a > b ? a : b; }

// Pages of 2^shift tokens that hold n >= 0 tokens.
MI355X_HD int64_t pages_of(int64_t n, int shift) { return (n + (int64_t(1) << shift) - 1) >> shift; }

// The request whose rows include row r (offsets ascend; n of them and the end),
// or -1.
MI355X_HD int seq_of_row(const int32_t *offsets, int n, int64_t r) {
    int lo = 0, hi = n;  // offsets[lo] <= r < offsets[hi], once the ends are checked
    if (n <= 0 || r < offsets[0] || r >= offsets[n]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Rows [first, first + n) of a request as its offsets give them, and the part
// [lo, hi) of 0 .. n that lies inside 0 .. n_rows.
struct SeqRows {
    int64_t first, n, lo, hi;
};
MI355X_HD SeqRows seq_rows(int64_t begin, int64_t end, int64_t n_rows) {
    SeqRows s;
    s.first = begin;
    s.n = idx_max(0, end - begin);
    s.lo = idx_min(s.n, idx_max(0, -begin));
    s.hi = idx_max(s.lo, idx_min(s.n, n_rows - begin));
    return s;
}

// Tokens [lo, hi) that the row at position pos sees, of `kv` cached ones of
// which the table's columns reach `reach`.
struct KeyRange {
    int64_t lo, hi;
};
MI355X_HD KeyRange visible_keys(int64_t pos, int64_t kv, int64_t reach, int window, bool causal) {
    KeyRange r;
    r.hi = idx_min(idx_max(kv, 0), reach);
    if (causal) r.hi = idx_min(r.hi, pos + 1);
    r.lo = window > 0 ? idx_max(0, pos - window + 1) : 0;
    r.hi = idx_max(r.hi, 0);
    r.lo = idx_min(r.lo, r.hi);
    return r;
}

// Whether a table entry names a page of the pool.
MI355X_HD bool page_in_pool(int32_t page, int64_t n_pages) { return page >= 0 && page < n_pages; }

// Whether a slot names a token's place in the pool.
MI355X_HD bool slot_in_pool(int64_t slot, int64_t n_pages, int shift) {
    return slot >= 0 && (slot >> shift) < n_pages;
}

}  // namespace mi355x
