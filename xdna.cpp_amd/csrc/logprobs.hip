// Log probabilities of given tokens, entropy and top tokens of rows of logits, in
// one pass over a row.
//
// With m the row's largest logit and d_i = scale (m - x_i) >= 0: S = sum exp(-d_i),
// log p_i = -d_i - log S, entropy = log S + sum exp(-d_i) d_i / S, every term of
// either sum of one sign.  The pass keeps S and E = sum 2^t t, t = -d log2 e, against
// the largest logit so far (2^(t) turns into 2^(t - shift) where a larger one comes).
//
// Top tokens.  The n-th largest of the threads' largest logits is no larger than
// the row's n-th largest, as each of them is a logit of its own: whatever is below it
// is no top token.  Logits that are not go into a list in LDS; the bound is raised
// when four times as many logits have been seen, so that about n log4 of the row's
// length get there.  A list that overflows (rows that ascend, many equal logits) is
// made again with the last bound, and failing that the row is searched n times: more than
// 1024 logits that are no smaller than the last top token's less 2^-7 of its size (what the
// bound is off by), as where all but a few have one finite value.
// That is right and slow: 2048 rows of 151936 in bf16 with 5, 20 and 64 top tokens 3.7, 11.9
// and 35 ms, one row 47, 160 and 606 us.  Masks of -inf are no candidates (119 us, and 14).
//
// Many rows, a workgroup each, are bound by memory: 2048 rows of 151936 in bf16, 622 MB,
// take 112 us (5.6 TB/s), with 5 top tokens 116, 20 128, 64 153.  One row in f32, 38 parts:
// 5.9 us, most of it a launch and a join, with 20 top tokens 10.2; 64 rows 12.6 and 19.8.
#include "far_parts.h"
#include "internal.h"
#include "paged_index.h"
#include "row_values.h"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace mi355x {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kLoads = 4;                         // of 8 logits that a thread has at a time
constexpr int kStep = 8 * kThreads;
constexpr int kBatch = kLoads * kStep;
constexpr int kList = 1024;
constexpr int kMostParts = 64;
constexpr int kMostItems = 1024;                  // parts of a call's rows
constexpr int kPartFloats = 4 + 2 * MI355X_LOGPROBS_MAX_TOP;
constexpr int kCounterStep = 32;                  // ints from one row's counter to the next: a cache line
constexpr size_t kCounterBytes = size_t(4) * kCounterStep * (kMostItems / 2);  // rows of two parts or more
// Top tokens up to which the bound is formed of 64 numbers, each the largest of a lane's
// logits in the four wavefronts, and not of all 256: fewer steps, a few more entries.
constexpr int kFewTop = 32;

struct LogitArgs {
    int64_t n_rows, stride;
    const void *logits;
    int n_vocab, n_tokens, n_top;
    float scale;
    int parts, part_len;  // of a row; part_len is a multiple of kStep
    FastDiv by_top;       // n_top, or 1
    const int32_t *tokens;
    float *token_logprobs, *entropy, *top_logprobs;
    int32_t *top_tokens;
    int *counters;  // 0 before and after a call
    float *ws;
};

// Numbers in the order of the logits (zeros have no sign), and of entries of a list:
// the larger logit, of equal ones the lower token, has the larger one.
__device__ __forceinline__ uint32_t rank_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t rank) {
    return __builtin_bit_cast(float, rank & 0x80000000u ? rank & 0x7FFFFFFFu : ~rank);
}
__device__ __forceinline__ uint64_t entry_of(float x, int at) {
    return static_cast<uint64_t>(rank_of(x)) << 32 | static_cast<uint32_t>(~at);
}
constexpr uint64_t kNoEntry = 0;  // below every entry

// A bound from below, 2^-7 of itself or less off, of the n-th largest of the 64 * N
// numbers that a wavefront's lanes hold: the 16 highest bits of its rank, found two by
// two.
template <int N>
__device__ __forceinline__ uint32_t nth_largest(const uint32_t *rank, int n) {
    uint32_t found = 0;
    for (int bit = 30; bit >= 16; bit -= 2) {
        int above[4];
#pragma unroll
        for (int t = 1; t < 4; ++t) {
            above[t] = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) above[t] += __builtin_popcountll(__ballot(rank[i] >= (found | static_cast<uint32_t>(t) << bit)));
        }
        found |= (above[3] >= n ? 3u : above[2] >= n ? 2u : above[1] >= n ? 1u : 0u) << bit;
    }
    return found;
}
// The logit of such a bound, but at least -FLT_MAX (below -inf lie NaN patterns).
__device__ __forceinline__ float bound_of(uint32_t rank) { return fmaxf(logit_of(rank), -FLT_MAX); }

// Sums against the largest logit so far, `high` (0 stands for it while it is -inf).
struct Sums {
    float high = -INFINITY, ref = 0.0f, s = 0.0f, e = 0.0f;
    // From now on against `to`, which is not below the logits that are in.
    __device__ __forceinline__ void raise(float to, float k) {
        if (!(to > high)) return;
        if (s != 0.0f) {
            // (a row's first logits may be the type's lowest value: the product may be infinite)
            const float shift = fmaxf((ref - to) * k, -1000.0f), f = __builtin_amdgcn_exp2f(shift);
            e = f * (e + shift * s);
            s *= f;
        }
        high = ref = to;
    }
    // Eight logits, added to each other first, so that no long chain of roundings grows.
    __device__ __forceinline__ void add8(const float *x, float k) {
        float s8 = 0.0f, e8 = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = (x[j] - ref) * k, p = __builtin_amdgcn_exp2f(t);
            s8 += p;                               // NaN where x is NaN or +inf
            e8 = fmaf(p, fmaxf(t, -1000.0f), e8);  // -inf adds nothing
        }
        s += s8;
        e += e8;
    }
};

struct Lds {
    uint64_t list[kList], best[kList];
    uint64_t top[MI355X_LOGPROBS_MAX_TOP];  // the top tokens in order
    int rank[64];
    float tops[2][kThreads];
    float sums[kWaves][2];
    int count, best_count, flag;
};

// Eight logits as floats, -inf behind the end.
template <int TYPE>
__device__ __forceinline__ void to_float(typename RowElem<TYPE>::Raw8 r, int i, int end, float *x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = static_cast<float>(r[j]);
    if (i + 8 > end) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j >= end) x[j] = -INFINITY;
    }
}

__device__ __forceinline__ void put(Lds &l, float x, int at) {
    const int p = atomicAdd(&l.count, 1);
    if (p < kList) l.list[p] = entry_of(x, at);
}

// The n first of `m` entries, in order, to l.top.  Up to 64 entries: each wavefront
// counts, for all of them, those of every kWaves-th that come before (l.rank is 0), and
// some may be none.
__device__ __forceinline__ int order(Lds &l, const uint64_t *list, int m, int n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (m <= 64) {
        const uint64_t x = lane < m ? list[lane] : kNoEntry;
        const int real = __builtin_popcountll(__ballot(x != kNoEntry));
        int r = 0;
#pragma unroll 4
        for (int q = wave; q < m; q += kWaves) r += list[q] > x;
        if (lane < m && r) atomicAdd(&l.rank[lane], r);
        __syncthreads();
        if (tid < m && l.rank[tid] < n) l.top[l.rank[tid]] = x;
        m = real;
    } else {
        for (int p = tid; p < m; p += kThreads) {
            const uint64_t x = list[p];
            int r = 0;
#pragma unroll 8
            for (int q = 0; q < m; ++q) r += list[q] > x;
            if (r < n) l.top[r] = x;
        }
    }
    __syncthreads();
    return min(m, n);
}

// The n first of the `count` entries of l.list, none of which has a rank below `bound()`.
// Called by all threads, with the list complete.
template <class F>
__device__ __forceinline__ int order_list(Lds &l, int count, int n, F bound) {
    if (count <= 64) return order(l, l.list, count, n);
    const uint32_t least = bound();
    if (threadIdx.x == 0) l.best_count = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < count; p += kThreads) {
        const uint64_t x = l.list[p];
        if (x != kNoEntry && x >> 32 >= least) l.best[atomicAdd(&l.best_count, 1)] = x;
    }
    __syncthreads();
    return order(l, l.best, l.best_count, n);
}

// The same by n searches of the row.
template <int TYPE>
__device__ int search(Lds &l, const void *row, int lo, int hi, int n) {
    typedef typename RowElem<TYPE>::T T;
    const T *p = static_cast<const T *>(row);
    const int tid = threadIdx.x;
    uint64_t last = ~uint64_t(0);
    int r = 0;
    for (; r < n; ++r) {
        uint64_t x = kNoEntry;
        for (int i = lo + tid; i < hi; i += kThreads) {
            const float v = static_cast<float>(p[i]);
            const uint64_t e = entry_of(v, i);
            if (v > -INFINITY && e < last && e > x) x = e;
        }
        __syncthreads();
        l.best[tid] = x;
        __syncthreads();
        for (int t = 0; t < kThreads; ++t) x = l.best[t] > x ? l.best[t] : x;
        if (x == kNoEntry) break;
        if (tid == 0) l.top[r] = x;
        last = x;
    }
    __syncthreads();
    return r;
}

// What a row's outputs are made of: its largest logit, the sums against it, and
// `found` top tokens in l.top.
template <int TYPE>
__device__ __forceinline__ void write_row(const LogitArgs &a, int64_t row, const Lds &l, float top, float s, float e,
                                          int found) {
    typedef typename RowElem<TYPE>::T T;
    const int tid = threadIdx.x;
    const bool bad = !(s < INFINITY), none = !bad && s == 0.0f;
    const float log_total = bad ? NAN : none ? 0.0f : logf(s);
    if (a.entropy && tid == 0)
        a.entropy[row] = bad ? NAN : none ? 0.0f : fmaf(-0.693147180559945309f, e / s, log_total);
    // in 64 bits: the difference of two f32 logits may pass f32's range where its multiple does not
    auto logprob = [&](float x) {
        return static_cast<float>(static_cast<double>(a.scale) * (static_cast<double>(x) - top) - log_total);
    };
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    for (int t = tid; t < a.n_tokens; t += kThreads) {
        const int token = a.tokens[row * a.n_tokens + t];
        const bool in = token >= 0 && token < a.n_vocab;
        const float x = in ? static_cast<float>(logits[token]) : 0.0f;
        a.token_logprobs[row * a.n_tokens + t] =
            bad || !in ? NAN : x == -INFINITY ? x : logprob(x);
    }
    for (int r = tid; r < a.n_top; r += kThreads) {
        const bool in = r < found && !bad;
        a.top_tokens[row * a.n_top + r] = in ? static_cast<int>(~static_cast<uint32_t>(l.top[r])) : -1;
        a.top_logprobs[row * a.n_top + r] =
            bad ? NAN : in ? logprob(logit_of(static_cast<uint32_t>(l.top[r] >> 32))) : -INFINITY;
    }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogitArgs a) {
    typedef typename RowElem<TYPE>::T T;
    typedef typename RowElem<TYPE>::Raw8 Raw8;
    __shared__ Lds l;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float k = a.scale * 1.44269504088896341f;
    const int n = a.n_top;
    for (int64_t item = blockIdx.x; item < a.n_rows * a.parts; item += gridDim.x) {
        const int64_t row = item / a.parts;
        const int part = static_cast<int>(item - row * a.parts);
        const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
        const int lo = part * a.part_len, hi = min(a.n_vocab, lo + a.part_len);
        Raw8 raw[kLoads];
        auto load = [&](int base) {
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
                if (base + c * kStep < hi) raw[c] = row_load8<TYPE>(logits, base + c * kStep + 8 * tid, hi);
        };
        load(lo);
        if (tid == 0) l.count = 0;
        if (tid < 64) l.rank[tid] = 0;
        Sums sums;
        float top = -INFINITY, bound = FLT_MAX;
        int turn = 0, next = 0;  // the bound is formed in batch `next`
        auto step = [&](int batch, int base, auto whole) {
            constexpr bool kWhole = decltype(whole)::value;  // the batch ends in the part
            auto in = [&](int c) { return kWhole || base + c * kStep < hi; };
            float x[kLoads][8], most = -INFINITY;
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
                if (in(c)) {
                    to_float<TYPE>(raw[c], kWhole ? INT_MIN : base + c * kStep + 8 * tid, hi, x[c]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) most = fmaxf(most, x[c][j]);
                }
            if (kWhole) load(base + kBatch);
            top = fmaxf(top, most);
            if (batch == next) {
                next = max(2, 4 * next);
                l.tops[turn][tid] = top;
                __syncthreads();
                float v[kWaves];
#pragma unroll
                for (int i = 0; i < kWaves; ++i) v[i] = l.tops[turn][64 * i + lane];
                turn ^= 1;
                const float of_lane = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                if (n > 0) {
                    uint32_t ranks[kWaves];
                    if (n <= kFewTop) {
                        ranks[0] = rank_of(of_lane);
                        bound = bound_of(nth_largest<1>(ranks, n));
                    } else {
#pragma unroll
                        for (int i = 0; i < kWaves; ++i) ranks[i] = rank_of(v[i]);
                        bound = bound_of(nth_largest<kWaves>(ranks, n));
                    }
                }
                sums.raise(wave_max(of_lane), k);
            }
            sums.raise(most, k);
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
                if (in(c)) sums.add8(x[c], k);
            if (most >= bound)
#pragma unroll
                for (int c = 0; c < kLoads; ++c)
                    if (in(c))
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (x[c][j] >= bound) put(l, x[c][j], base + c * kStep + 8 * tid + j);
        };
        int batch = 0, base = lo;
        for (; base + kBatch <= hi; base += kBatch, ++batch) step(batch, base, std::true_type{});
        if (base < hi) step(batch, base, std::false_type{});
        // the workgroup's sums, and the n-th largest of what its threads had
        l.tops[turn][tid] = top;
        __syncthreads();
        float v[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v[i] = l.tops[turn][64 * i + lane];
        const float all = wave_max(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
        sums.raise(all, k);
        const float ws = wave_sum(sums.s), we = wave_sum(sums.e);
        if (lane == 0) {
            l.sums[wave][0] = ws;
            l.sums[wave][1] = we;
        }
        int found = 0, count = l.count;
        if (n > 0) {
            auto last_bound = [&]() {
                uint32_t ranks[kWaves];
#pragma unroll
                for (int i = 0; i < kWaves; ++i) ranks[i] = rank_of(v[i]);
                return nth_largest<kWaves>(ranks, n);
            };
            if (count > kList) {  // once more, with the bound that the whole row gives
                bound = bound_of(last_bound());
                __syncthreads();
                if (tid == 0) l.count = 0;
                __syncthreads();
                for (int i = lo + tid; i < hi; i += kThreads) {
                    const float x = static_cast<float>(logits[i]);
                    if (x >= bound) put(l, x, i);
                }
                __syncthreads();
                count = l.count;
            }
            found = count > kList ? search<TYPE>(l, logits, lo, hi, n) : order_list(l, count, n, last_bound);
        } else {
            __syncthreads();
        }
        float s = 0.0f, e = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            s += l.sums[w][0];
            e += l.sums[w][1];
        }
        if (a.parts == 1) {
            write_row<TYPE>(a, row, l, all, s, e, found);
        } else {
            const FarParts far(a.ws);
            const int at = static_cast<int>(item) * kPartFloats;
            if (tid == 0) far.store4(at, f32x4{all, s, e, 0.0f});
            for (int r = tid; r < n; r += kThreads)
                far.store2(at + 4 + 2 * r, __builtin_bit_cast(u32x2_a, r < found ? l.top[r] : kNoEntry));
            if (last_of(a.counters + kCounterStep * row, a.parts, &l.flag)) {
                const int first = static_cast<int>(row) * a.parts, total = a.parts * n;  // at most kList
                f32x4 p = {-INFINITY, 0.0f, 0.0f, 0.0f};  // the row's parts, one a lane
                if (lane < a.parts) p = far.load4((first + lane) * kPartFloats);
                uint64_t entry[kList / kThreads];  // all on their way before one is waited for
#pragma unroll
                for (int i = 0; i < kList / kThreads; ++i) {
                    const int j = min(i * kThreads + tid, total - 1), q = divided(j, a.by_top);
                    entry[i] = kNoEntry;
                    if (i * kThreads < total)
                        entry[i] = __builtin_bit_cast(uint64_t, far.load2((first + q) * kPartFloats + 4 + 2 * (j - q * n)));
                }
#pragma unroll
                for (int i = 0; i < kList / kThreads; ++i)
                    if (i * kThreads + tid < total) l.list[i * kThreads + tid] = entry[i];
                if (tid < 64) l.rank[tid] = 0;
                const float most = wave_max(p[0]);
                Sums mine;
                mine.high = mine.ref = p[0];  // (not used where it is -inf: the sums are 0)
                mine.s = p[1];
                mine.e = p[2];
                mine.raise(most, k);
                const float ts = wave_sum(mine.s), te = wave_sum(mine.e);
                __syncthreads();
                if (n > 0)
                    found = order_list(l, total, n, [&]() {
                        // the n-th largest of the first of each part, or of its first few
                        uint32_t ranks[kWaves];
                        if (2 * n <= a.parts + 8) {
                            ranks[0] = lane < a.parts ? static_cast<uint32_t>(l.list[lane * n] >> 32) : 0;
                            return nth_largest<1>(ranks, n);
                        }
                        const int few = min(n, kThreads / a.parts);
#pragma unroll
                        for (int i = 0; i < kWaves; ++i) {
                            const int j = 64 * i + lane, q = j / few;
                            ranks[i] = q < a.parts ? static_cast<uint32_t>(l.list[q * n + j - q * few] >> 32) : 0;
                        }
                        return nth_largest<kWaves>(ranks, n);
                    });
                write_row<TYPE>(a, row, l, most, ts, te, found);
            }
        }
        __syncthreads();  // l
    }
}

template <int TYPE>
int launch_type(mi355x_ctx *ctx, const LogitArgs &a) {
    const int64_t groups = std::min<int64_t>(a.n_rows * a.parts, 1 << 20);
    logprobs_kernel<TYPE><<<static_cast<unsigned>(groups), kThreads, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace

size_t logprobs_workspace_bytes(const mi355x_ctx *) {
    return kCounterBytes + size_t(4) * kMostItems * kPartFloats;
}

int launch_logprobs(mi355x_ctx *ctx, const mi355x_logprobs_args &u) {
    LogitArgs a{};
    a.n_rows = u.n_rows;
    a.stride = u.stride;
    a.logits = u.logits;
    a.n_vocab = u.n_vocab;
    a.n_tokens = u.n_tokens;
    a.n_top = u.n_top;
    a.by_top = fast_div(static_cast<uint32_t>(std::max(u.n_top, 1)));
    a.scale = u.scale;
    a.tokens = u.tokens;
    a.token_logprobs = u.token_logprobs;
    a.entropy = u.entropy;
    a.top_logprobs = u.top_logprobs;
    a.top_tokens = u.top_tokens;
    a.counters = static_cast<int *>(u.workspace);
    a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(u.workspace) + kCounterBytes);
    // Few rows are cut into parts of half a batch or more, so that a part is one round of loads
    // (one row of 151936 with 20 top tokens in parts of 4096 10.2 us, of 8192 11.6), as many
    // as 4 workgroups a CU, or 3 with 32 bits, of which twice as much is under way (3, 4 and 8 a
    // CU: 64 rows of 151936 in f32 19.8, 24.7, 27.6, in bf16 17.5, 16.8, 20.3; 400 of 50000 in f32
    // 22, 32; 300 of 151936 in bf16 39, 35, 42).
    const int items = std::min(kMostItems, (u.type == MI355X_TYPE_F32 ? 3 : 4) * ctx->num_cus);
    int64_t parts = std::min<int64_t>(items / u.n_rows, (u.n_vocab + kBatch / 2 - 1) / (kBatch / 2));
    parts = std::min<int64_t>(parts, std::min(kMostParts, kList / std::max(u.n_top, 1)));
    parts = std::max<int64_t>(parts, 1);
    a.part_len = static_cast<int>((u.n_vocab + kStep * parts - 1) / (kStep * parts) * kStep);
    a.parts = static_cast<int>((u.n_vocab + a.part_len - 1) / a.part_len);
    if (u.type == MI355X_TYPE_F32) return launch_type<MI355X_TYPE_F32>(ctx, a);
    if (u.type == MI355X_TYPE_F16) return launch_type<MI355X_TYPE_F16>(ctx, a);
    return launch_type<MI355X_TYPE_BF16>(ctx, a);
}

}  // namespace mi355x
