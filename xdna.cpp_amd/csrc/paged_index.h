// Index arithmetic of the paged KV cache, shared by the kernels and by the CPU
// tests (no HIP in here but the function attributes).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define MI355X_HD __attribute__((host)) __attribute__((device)) inline __attribute__((always_inline))
#else
#define MI355X_HD inline
#endif

namespace mi355x {

MI355X_HD int64_t idx_min(int64_t a, int64_t b) { return a < b ? a : b; }
MI355X_HD int64_t idx_max(int64_t a, int64_t b) { return a > b ? a : b; }

// n / d for 0 <= n < 2^31 as a product and a shift (d >= 1): mul = floor(2^(31 +
// l) / d) + 1 with l = ceil(log2 d) is above 2^(31 + l) / d by at most 2^l parts
// of its d, which moves no quotient of n < 2^31.
struct FastDiv {
    uint32_t d, mul, shift;
};
MI355X_HD FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 31};
    while ((uint64_t(1) << (f.shift - 31)) < d) ++f.shift;
    f.mul = static_cast<uint32_t>((uint64_t(1) << f.shift) / d + 1);
    return f;
}
MI355X_HD int32_t divided(int32_t n, const FastDiv &f) {
    return static_cast<int32_t>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * f.mul) >> f.shift);
}

// a / b, by 32-bit division where both fit (64-bit division is long on the GPU).
MI355X_HD int64_t quotient(int64_t a, int64_t b) {
    if (((static_cast<uint64_t>(a) | static_cast<uint64_t>(b)) >> 32) == 0)
        return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// `total` units in `groups` stretches of equal length, the first of them one longer.
struct Stretches {
    int64_t total, each, longer;
    int groups;
};
MI355X_HD Stretches stretches(int64_t total, int groups) {
    Stretches s;
    s.total = total;
    s.groups = groups;
    s.each = quotient(total, groups);
    s.longer = total - s.each * groups;
    return s;
}
MI355X_HD int64_t stretch_begin(const Stretches &s, int64_t g) { return s.each * g + idx_min(g, s.longer); }
// The stretch that has unit u < total.
MI355X_HD int64_t stretch_of(const Stretches &s, int64_t u) {
    const int64_t lead = s.longer * (s.each + 1);
    return u < lead ? quotient(u, s.each + 1) : s.longer + quotient(u - lead, s.each);
}

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
