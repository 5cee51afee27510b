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
// made again with the last bound, and failing that the row is searched n times.
#include "far_parts.h"
#include "internal.h"
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
constexpr size_t kCounterBytes = 4 * kMostItems;

struct LogitArgs {
    int64_t n_rows, stride;
    const void *logits;
    int n_vocab, n_tokens, n_top;
    float scale;
    int parts, part_len;  // of a row; part_len is a multiple of 8
    const int32_t *tokens;
    float *token_logprobs, *entropy, *top_logprobs;
    int32_t *top_tokens;
    int *counters;  // 0 before and after a call
    float *ws;
};

// The larger logit first, of equal ones the lower token.
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

// A bound from below, at least -FLT_MAX and 2^-11 of itself or less off, of the n-th
// largest of the 64 * N numbers that a wavefront's lanes hold: the 20 highest bits of
// it, found one by one.
template <int N>
__device__ __forceinline__ float nth_largest(const float *v, int n) {
    uint32_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[i] + 0.0f);  // no zero with a sign
        key[i] = b & 0x80000000u ? ~b : b | 0x80000000u;               // in the order of the numbers
    }
    uint32_t found = 0;
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t tried = found | 1u << bit;
        int above = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) above += __builtin_popcountll(__ballot(key[i] >= tried));
        if (above >= n) found = tried;
    }
    const uint32_t b = found & 0x80000000u ? found & 0x7FFFFFFFu : ~found;
    return fmaxf(__builtin_bit_cast(float, b), -FLT_MAX);  // below -inf lie NaN patterns
}

// Sums against the largest logit so far, `high` (0 stands for it while it is -inf).
struct Sums {
    float high = -INFINITY, ref = 0.0f, s = 0.0f, e = 0.0f;
    // From now on against `to`, which is not below the logits that are in.
    __device__ __forceinline__ void raise(float to, float k) {
        if (!(to > high)) return;
        if (s != 0.0f) {
            const float shift = (ref - to) * k, f = __builtin_amdgcn_exp2f(shift);
            e = f * (e + shift * s);
            s *= f;
        }
        high = ref = to;
    }
    __device__ __forceinline__ void add(float x, float k) {
        const float t = (x - ref) * k, p = __builtin_amdgcn_exp2f(t);
        s += p;                              // NaN where x is NaN or +inf
        e = fmaf(p, fmaxf(t, -1000.0f), e);  // -inf adds nothing
    }
};

struct Lds {
    float list[kList];
    int list_at[kList];
    float best[kList];
    int best_at[kList];
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
    if (p < kList) {
        l.list[p] = x;
        l.list_at[p] = at;
    }
}

// The n top entries of the `count` ones in l.list that are not below `bound`, in
// order, to l.best; how many there are.  Called by all threads, with the list
// complete.
__device__ __forceinline__ int order_list(Lds &l, int count, float bound, int n) {
    const int tid = threadIdx.x;
    if (tid == 0) l.best_count = 0;
    __syncthreads();
    for (int p = tid; p < count; p += kThreads)
        if (l.list[p] >= bound) {
            const int q = atomicAdd(&l.best_count, 1);
            l.best[q] = l.list[p];
            l.best_at[q] = l.list_at[p];
        }
    __syncthreads();
    const int m = l.best_count;
    for (int p = tid; p < m; p += kThreads) {
        const float x = l.best[p];
        const int at = l.best_at[p];
        int r = 0;
        for (int q = 0; q < m; ++q) r += before(l.best[q], l.best_at[q], x, at);
        if (r < n) {
            l.list[r] = x;
            l.list_at[r] = at;
        }
    }
    __syncthreads();
    return min(m, n);
}

// The same by n searches of the row.
template <int TYPE>
__device__ int search(Lds &l, const void *row, int lo, int hi, int n) {
    typedef typename RowElem<TYPE>::T T;
    const T *p = static_cast<const T *>(row);
    const int tid = threadIdx.x;
    float last = INFINITY;
    int last_at = -1, r = 0;
    for (; r < n; ++r) {
        float x = -INFINITY;
        int at = INT_MAX;
        for (int i = lo + tid; i < hi; i += kThreads) {
            const float v = static_cast<float>(p[i]);
            if (v > -INFINITY && before(last, last_at, v, i) && before(v, i, x, at)) {
                x = v;
                at = i;
            }
        }
        __syncthreads();
        l.best[tid] = x;
        l.best_at[tid] = at;
        __syncthreads();
        for (int t = 0; t < kThreads; ++t)
            if (before(l.best[t], l.best_at[t], x, at)) {
                x = l.best[t];
                at = l.best_at[t];
            }
        if (at == INT_MAX) break;
        if (tid == 0) {
            l.list[r] = x;
            l.list_at[r] = at;
        }
        last = x;
        last_at = at;
    }
    __syncthreads();
    return r;
}

// What a row's outputs are made of: its largest logit, the sums against it, and
// `found` top tokens in l.list.
template <int TYPE>
__device__ __forceinline__ void write_row(const LogitArgs &a, int64_t row, const Lds &l, float top, float s, float e,
                                          int found) {
    typedef typename RowElem<TYPE>::T T;
    const int tid = threadIdx.x;
    const bool bad = !(s < INFINITY), none = !bad && s == 0.0f;
    const float log_total = bad ? NAN : none ? 0.0f : logf(s);
    if (a.entropy && tid == 0)
        a.entropy[row] = bad ? NAN : none ? 0.0f : fmaf(-0.693147180559945309f, e / s, log_total);
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    for (int t = tid; t < a.n_tokens; t += kThreads) {
        const int token = a.tokens[row * a.n_tokens + t];
        const bool in = token >= 0 && token < a.n_vocab;
        const float x = in ? static_cast<float>(logits[token]) : 0.0f;
        a.token_logprobs[row * a.n_tokens + t] =
            bad || !in ? NAN : x == -INFINITY ? x : a.scale * (x - top) - log_total;
    }
    for (int r = tid; r < a.n_top; r += kThreads) {
        const bool in = r < found && !bad;
        a.top_tokens[row * a.n_top + r] = in ? l.list_at[r] : -1;
        a.top_logprobs[row * a.n_top + r] = bad ? NAN : in ? a.scale * (l.list[r] - top) - log_total : -INFINITY;
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
            for (int c = 0; c < kLoads; ++c) raw[c] = row_load8<TYPE>(logits, base + c * kStep + 8 * tid, hi);
        };
        load(lo);
        if (tid == 0) l.count = 0;
        Sums sums;
        float top = -INFINITY, bound = FLT_MAX;
        int turn = 0, next = 0;  // the bound is formed in batch `next`
        for (int batch = 0, base = lo; base < hi; base += kBatch, ++batch) {
            float x[kLoads][8], most = -INFINITY;
#pragma unroll
            for (int c = 0; c < kLoads; ++c) to_float<TYPE>(raw[c], base + c * kStep + 8 * tid, hi, x[c]);
            if (base + kBatch < hi) load(base + kBatch);
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, x[c][j]);
            top = fmaxf(top, most);
            if (batch == next) {
                next = max(2, 4 * next);
                l.tops[turn][tid] = top;
                __syncthreads();
                float v[kWaves];
#pragma unroll
                for (int i = 0; i < kWaves; ++i) v[i] = l.tops[turn][64 * i + lane];
                turn ^= 1;
                if (n > 0) bound = nth_largest<kWaves>(v, n);
                sums.raise(wave_max(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))), k);
            }
            sums.raise(most, k);
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) sums.add(x[c][j], k);
            if (most >= bound)
#pragma unroll
                for (int c = 0; c < kLoads; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (x[c][j] >= bound) put(l, x[c][j], base + c * kStep + 8 * tid + j);
        }
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
            bound = nth_largest<kWaves>(v, n);
            if (count > kList) {  // once more, with the bound that the whole row gives
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
            found = count > kList ? search<TYPE>(l, logits, lo, hi, n) : order_list(l, count, bound, n);
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
            for (int r = tid; r < n; r += kThreads) {
                far.store(at + 4 + r, r < found ? l.list[r] : -INFINITY);
                far.store(at + 4 + MI355X_LOGPROBS_MAX_TOP + r,
                          __builtin_bit_cast(float, r < found ? l.list_at[r] : -1));
            }
            if (last_of(a.counters + row, a.parts, &l.flag)) {
                // the row's parts, one a lane
                const int first = static_cast<int>(row) * a.parts;
                f32x4 p = {-INFINITY, 0.0f, 0.0f, 0.0f};
                if (lane < a.parts) p = far.load4((first + lane) * kPartFloats);
                const float most = wave_max(p[0]);
                Sums mine;
                mine.high = mine.ref = p[0];  // (not used where it is -inf: the sums are 0)
                mine.s = p[1];
                mine.e = p[2];
                mine.raise(most, k);
                const float ts = wave_sum(mine.s), te = wave_sum(mine.e);
                if (n > 0) {
                    const int total = a.parts * n;  // at most kList
                    for (int j = tid; j < total; j += kThreads) {
                        const int q = j / n, from = (first + q) * kPartFloats + 4 + j - q * n;
                        l.list[j] = far.load(from);
                        l.list_at[j] = __builtin_bit_cast(int, far.load(from + MI355X_LOGPROBS_MAX_TOP));
                    }
                    __syncthreads();
                    float c[kList / 64];
#pragma unroll
                    for (int i = 0; i < kList / 64; ++i)
                        c[i] = 64 * i + lane < total ? l.list[64 * i + lane] : -INFINITY;
                    bound = nth_largest<kList / 64>(c, n);
                    found = order_list(l, total, bound, n);
                }
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
    a.scale = u.scale;
    a.tokens = u.tokens;
    a.token_logprobs = u.token_logprobs;
    a.entropy = u.entropy;
    a.top_logprobs = u.top_logprobs;
    a.top_tokens = u.top_tokens;
    a.counters = static_cast<int *>(u.workspace);
    a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(u.workspace) + kCounterBytes);
    // few rows are cut into parts of half a batch or more
    int64_t parts = std::min<int64_t>(kMostItems / u.n_rows, (u.n_vocab + kBatch / 2 - 1) / (kBatch / 2));
    parts = std::min<int64_t>(parts, std::min(kMostParts, kList / std::max(u.n_top, 1)));
    parts = std::max<int64_t>(parts, 1);
    a.part_len = static_cast<int>((u.n_vocab + 8 * parts - 1) / (8 * parts) * 8);
    a.parts = static_cast<int>((u.n_vocab + a.part_len - 1) / a.part_len);
    if (u.type == MI355X_TYPE_F32) return launch_type<MI355X_TYPE_F32>(ctx, a);
    if (u.type == MI355X_TYPE_F16) return launch_type<MI355X_TYPE_F16>(ctx, a);
    return launch_type<MI355X_TYPE_BF16>(ctx, a);
}

}  // namespace mi355x
