// Device-side building blocks of the attention kernels.
#pragma once

#include "paged_index.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "mi355x-attention.h"

namespace mi355x {

// A call as the kernels see it.
struct AttnArgs {
    const void *q, *k, *v;
    const int32_t *row_offsets, *kv_lens, *table;
    void *out;
    float *ws;      // parts
    int *counters;  // 0 before and after a call
    int64_t q_stride, out_stride, table_stride;
    int64_t head_stride;
    int64_t n_rows;
    uint32_t page_stride, token_stride;
    int reach;          // tokens that the table's columns hold, at most 2^30
    int row_limit;      // requests of at most (token form) or more than (chunk form) so many head rows
    float scale2;            // scale log2 e: scores are in factors of 2
    float cap_in, cap_out;   // 2 scale log2 e / softcap (finite) and softcap log2 e; 0: no cap
    float line_share;  // token form: 1 / (12 teams of a join x requests x KV heads)
    FastDiv group;  // query heads of a KV head
    int n_seqs, n_kv_heads;
    int n_pages, shift, window, causal, f32_out;
    int split;    // chunk form: parts of an item's keys
    int by_page;  // the rows of a load into LDS share a page, with 32-bit offsets in it
};

constexpr float kLog2e = 1.44269504088896341f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_a __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_a __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// The pool's 16-bit type: matrix products, roundings, the bits of its exponent
// (all set: infinity or NaN), and by how many factors of 2 weights are held above
// 2^(s - m) (see Reference).
template <int TYPE>
struct Num;
template <>
struct Num<MI355X_TYPE_F16> {
    typedef _Float16 T;
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kExp = 0x7C00u;
    static constexpr float kRaise = 7.0f;
    static __device__ __forceinline__ f32x4 mfma16(V8 a, V8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Num<MI355X_TYPE_BF16> {
    typedef __bf16 T;
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kExp = 0x7F80u;
    static constexpr float kRaise = 0.0f;
    static __device__ __forceinline__ f32x4 mfma16(V8 a, V8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// Whether any of the eight 16-bit values is an infinity or a NaN.
template <int TYPE>
__device__ __forceinline__ bool not_finite(u32x4_a v) {
    constexpr uint32_t e = Num<TYPE>::kExp;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (v[i] & e) == e || ((v[i] >> 16) & e) == e;
    return bad;
}

// Four rows of one column each from a 4-row x 16-column block of 16-bit values
// per 16 lanes: lane c of the 16 passes the address of 4 values of row c / 4
// from column 4 (c % 4) on, and gets column c of the four rows.
// __restrict__ keeps the compiler from taking every LDS load that is on its way
// (global_load_lds) for a write to the same place, and waiting for it: the
// kernels' barriers order those.
__device__ __forceinline__ u32x2_a lds_read_transposed(const s16x4 *__restrict__ p) {
    return __builtin_bit_cast(
        u32x2_a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p)));
}

// 16 bytes per lane from memory to LDS, lane after lane from `to` on.
__device__ __forceinline__ void load_lds16(const void *from, unsigned char *to) {
    __builtin_amdgcn_global_load_lds(
        reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(reinterpret_cast<uintptr_t>(from)),
        (__attribute__((address_space(3))) uint32_t *)(to), 16, 0, 0);
}

// Scores of N values x of q . k, in factors of 2.  tanh y as 1 - 2 / (1 + e^2y),
// within 2^-23 of 1, and below 1/8, where that is too coarse for a small score,
// by its series (the next term is 62/2835 y^8: 2^-29).
template <int N>
__device__ __forceinline__ void scores2(float (&x)[N], const AttnArgs &a) {
    if (a.cap_out == 0.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= a.scale2;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float e = x[i] * a.cap_in, y = e * (0.5f / kLog2e), y2 = y * y;
            const float small = x[i] * a.scale2 *
                                fmaf(y2, fmaf(y2, fmaf(y2, -17.0f / 315, 2.0f / 15), -1.0f / 3), 1.0f);
            const float big = fmaf(-2.0f * a.cap_out, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e)), a.cap_out);
            x[i] = fabsf(y) < 0.125f ? small : big;
        }
    }
}

// Maximum and sum over a lane and the one 32 lanes on.
__device__ __forceinline__ void both_halves(float v, float *a, float *b) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t x = r[0], y = r[1];
    *a = __builtin_bit_cast(float, x);
    *b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float half_max(float v) {
    float a, b;
    both_halves(v, &a, &b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
    float a, b;
    both_halves(v, &a, &b);
    return a + b;
}

// Maximum and sum over the four lanes with the same number modulo 16.
__device__ __forceinline__ void both_rows(float v, float *a, float *b) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    const uint32_t x = r[0], y = r[1];
    *a = __builtin_bit_cast(float, x);
    *b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float quad_max(float v) {
    float a, b;
    both_rows(v, &a, &b);
    return half_max(fmaxf(a, b));
}
__device__ __forceinline__ float quad_sum(float v) {
    float a, b;
    both_rows(v, &a, &b);
    return half_sum(a + b);
}

// What a row's sums are held relative to: weights are 2^(s - m + kRaise).  A tile's
// largest score may be above m by kSlack (in factors of 2) before m moves there and the
// sums are scaled.  Each row moves by its own scores alone, also where another row of
// its wavefront does: tokens that it does not see leave its roundings as they are.
//
// bf16 weights are as exact at any size, so their m only rises.  f16 weights are exact
// to half a step down to 2^-14 and have steps of 2^-24 below: behind one token that
// takes nearly all of the weight, others of 2^-25 of it would be lost, however much
// they add up to.  So f16's m also falls, to the largest score of a tile that is all
// further below: the largest weight of a tile lies between 2^-1 and 2^15 wherever it
// comes.  m falls by no more than kMostFall below its highest, which the f32 sums
// hold; smaller weights are lost in them.  (Costs 0 to 2%: f16 chunk of 512 tokens
// 44.7 -> 45.3 us, prompt of 8192 632 -> 634, 64 ragged requests 212.)
constexpr float kSlack = 8.0f, kMostFall = 40.0f;

__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.0f : m; }

template <int TYPE>
struct Reference {
    static constexpr bool kFalls = Num<TYPE>::kRaise > 0.0f;
    float m = -INFINITY, least = -INFINITY;

    // Whether a tile whose largest score is `top` moves it.
    __device__ __forceinline__ bool moves(float top) const {
        if (!kFalls) return top > m + kSlack || (m == -INFINITY && top > m);
        return fabsf(top - m) > kSlack && top > -INFINITY && (top > m || m > least);
    }
    // Moves it there, if so; the factor that the row's sums take.
    __device__ __forceinline__ float move(bool there, float top) {
        const float to = there ? kFalls ? fmaxf(top, least) : top : m, keep = __builtin_amdgcn_exp2f(m - finite_base(to));
        m = to;
        if (kFalls) least = fmaxf(least, m - kMostFall);
        return keep;
    }
    // What scores are taken relative to.
    __device__ __forceinline__ float base() const { return finite_base(m) - Num<TYPE>::kRaise; }
};

// A weight meets v as a sum of 16-bit planes.  For an f32 output as many as leave no
// more than 2^-22 of it: two of f16, three of bf16, of which two leave 2^-16 (errors of up to
// 2e-6 of the norm against 64 bits where f32 weights give 5e-7; the third takes a chunk of
// 512 tokens on 4096 from 44 to 51 us, a prompt of 4096 from 217 to 275, single tokens
// nothing).  For a 16-bit output one in the chunk form, which the matrix and vector units
// bound, since the output's own rounding is as large (bf16: 2.1e-3 of the norm, 1.65e-3
// with f32 weights), and two in the token form, where the matrix cores idle.
constexpr int f32_planes(int type) { return type == MI355X_TYPE_BF16 ? 3 : 2; }

// The planes of weight i.
template <int TYPE, int PLANES>
__device__ __forceinline__ void split_weight(float p, typename Num<TYPE>::V8 (&w)[PLANES], int i) {
#pragma unroll
    for (int k = 0; k < PLANES; ++k) {
        const typename Num<TYPE>::T h = static_cast<typename Num<TYPE>::T>(p);
        w[k][i] = h;
        if (k + 1 < PLANES) p -= static_cast<float>(h);
    }
}

// Rows and tokens of a request.
struct SeqGeo {
    int64_t first;    // its first row
    int64_t tok_lo;   // its tokens tok_lo .. tok_lo + n_tok - 1 have rows inside the call's
    int n_tok;
    int rows;         // n_tok * group: one row per token and query head of a KV head
    int64_t pos0;     // position of token 0
    int64_t kv;
};

__device__ __forceinline__ SeqGeo seq_geo(const AttnArgs &a, int32_t begin, int32_t end, int32_t kv) {
    const SeqRows r = seq_rows(begin, end, a.n_rows);
    SeqGeo g;
    g.first = r.first;
    g.tok_lo = r.lo;
    g.n_tok = static_cast<int>(r.hi - r.lo);
    g.rows = g.n_tok * static_cast<int>(a.group.d);
    g.kv = kv;
    g.pos0 = g.kv - r.n;
    return g;
}

__device__ __forceinline__ SeqGeo seq_geo(const AttnArgs &a, int s) {
    return seq_geo(a, a.row_offsets[s], a.row_offsets[s + 1], a.kv_lens[s]);
}

// Tokens lo .. hi - 1 (at most 2^30) that a token of the request sees.
struct Keys {
    int lo, hi;
};
__device__ __forceinline__ Keys token_keys(const AttnArgs &a, const SeqGeo &g, int64_t token) {
    const KeyRange r = visible_keys(g.pos0 + token, g.kv, a.reach, a.window, a.causal != 0);
    return Keys{static_cast<int>(r.lo), static_cast<int>(r.hi)};
}

// Where a token lies behind its KV head's first value; page in the pool.
__device__ __forceinline__ int64_t token_at(const AttnArgs &a, int page, int key) {
    const uint32_t in_page = static_cast<uint32_t>(key) & ((1u << a.shift) - 1);
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * a.page_stride +
                                static_cast<uint64_t>(in_page) * a.token_stride);
}

// Which of the BITS keys from `base` on lie in [lo, hi), a bit each.
template <typename MASK>
__device__ __forceinline__ MASK range_mask(int lo, int hi, int base) {
    constexpr int kBits = 8 * sizeof(MASK);
    const int l = max(lo - base, 0), h = min(hi - base, kBits);
    return h > l ? static_cast<MASK>(static_cast<MASK>(~MASK(0) >> (kBits - h)) & ~((MASK(1) << l) - 1)) : MASK(0);
}

// Four values of a row's output.
template <int TYPE>
__device__ __forceinline__ void store_out4(const AttnArgs &a, int64_t at, f32x4 v) {
    typedef typename Num<TYPE>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (a.f32_out) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + at) = v;
    } else {
        T4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = static_cast<T>(v[i]);
        *reinterpret_cast<T4 *>(static_cast<T *>(a.out) + at) = h;
    }
}

// Where the output of head row `row` of KV head kvh begins.
__device__ __forceinline__ int64_t out_at(const AttnArgs &a, const SeqGeo &g, int kvh, int row, int hd) {
    const int token = divided(row, a.group), group = static_cast<int>(a.group.d);
    const int64_t head = static_cast<int64_t>(kvh) * group + (row - token * group);
    return (g.first + g.tok_lo + token) * a.out_stride + head * hd;
}

// Parts of a row's sums that travel between workgroups of one launch, whose dies'
// L2s do not see each other: stored and read past them, so that no L2 has to be
// written back or emptied (fences that do so made 64 ragged requests 454 us
// instead of 196).  A workgroup that has waited for its stores and met a barrier
// may then count itself in.
constexpr int kPastL2 = 16;  // the sc1 bit of a buffer operation
struct FarParts {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ explicit FarParts(float *base)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0xFFFFFFFFu, kBufferWord3)) {}
    __device__ __forceinline__ void store(int at, float v) const {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rsrc, 4 * at, 0, kPastL2);
    }
    __device__ __forceinline__ void store4(int at, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_a, v), rsrc, 4 * at, 0, kPastL2);
    }
    __device__ __forceinline__ float load(int at) const {
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, 4 * at, 0, kPastL2));
    }
    __device__ __forceinline__ f32x4 load4(int at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, 4 * at, 0, kPastL2));
    }
};
// The same of an earlier launch.
struct NearParts {
    const float *base;
    __device__ __forceinline__ explicit NearParts(const float *b) : base(b) {}
    __device__ __forceinline__ float load(int at) const { return base[at]; }
    __device__ __forceinline__ f32x4 load4(int at) const { return *reinterpret_cast<const f32x4 *>(base + at); }
};

// Counts this workgroup in at *counter, which `n` of them do; true for the last
// one, which finds the others' parts complete and leaves the counter at 0.
// Called by all threads; `flag` is LDS.
__device__ __forceinline__ bool last_of(int *counter, int n, int *flag) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's stores
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == n - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = before == n - 1;
    }
    __syncthreads();
    return *flag != 0;
}

// Sums of 4 values of a row over some of its parts.
struct Joined {
    float top = -INFINITY, den = 0.0f;
    f32x4 num = {0, 0, 0, 0};
    __device__ __forceinline__ void add(float m, float l, f32x4 x) {
        const float t = fmaxf(top, m), ref = finite_base(t);
        const float f = __builtin_amdgcn_exp2f(top - ref), h = __builtin_amdgcn_exp2f(m - ref);
        num = num * f + x * h;
        den = den * f + l * h;
        top = t;
    }
    __device__ __forceinline__ f32x4 value() const {
        return den == 0.0f ? f32x4{0, 0, 0, 0} : num * (1.0f / den);
    }
};

// Adds parts first, first + step, .. below n: part i has the row's 4 values at
// values(i), its maximum at maximum(i) and its sum at total(i) of `parts`.  The
// loads of eight parts go out together.
template <typename P, typename V, typename M, typename L>
__device__ __forceinline__ void join_parts(Joined &j, const P &parts, int n, int first, int step, V values, M maximum,
                                           L total) {
    for (int i = first; i < n; i += 8 * step) {
        f32x4 x[8];
        float m[8], l[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int p = min(i + k * step, n - 1);
            x[k] = parts.load4(values(p));
            m[k] = parts.load(maximum(p));
            l[k] = parts.load(total(p));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k * step < n) j.add(m[k], l[k], x[k]);
    }
}

// A value that all lanes share, told to the compiler as such.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Exclusive scan of one value per thread over a workgroup of WAVES wavefronts;
// *total is the sum.  `tmp` holds WAVES values and is free after the call's
// last barrier.
template <int WAVES>
__device__ __forceinline__ int64_t group_scan(int64_t v, int64_t *tmp, int64_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(in, d);
        if (lane >= d) in += u;
    }
    if (lane == 63) tmp[wave] = in;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += tmp[w];
        sum += tmp[w];
    }
    __syncthreads();
    *total = sum;
    return before + in - v;
}

// The chunk form (paged_attention_chunk.hip): requests of more than
// a.row_limit head rows, and its part of the workspace.
int launch_attention_chunk(mi355x_ctx *ctx, const AttnArgs &a, int type, int head_dim);
size_t attention_chunk_workspace(const mi355x_ctx *ctx, int head_dim);

}  // namespace mi355x
