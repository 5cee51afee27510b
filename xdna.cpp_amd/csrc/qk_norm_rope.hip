// Bias, norms of query and key heads, rotation, and the store of keys and
// values into cache pages, in one pass.
//
// Per row and head: x = in + bias; x *= norm / sqrt(mean(x^2) + eps); pairs
// turned by angle = position * inv_freq.  Every value is read once and written
// once and takes a few operations, so HBM bounds long calls and latency short
// ones.  The angle is formed in 64 bits (a position of 10^6 times a frequency
// of 1 has an f32 step of 0.06 rad), reduced to a fraction of a turn there, and
// its sine and cosine taken in f32.
#include "internal.h"
#include "paged_index.h"

#include <algorithm>

namespace mi355x {
namespace {

struct RopeArgs {
    int64_t n_rows;
    int n_heads, n_kv_heads, head_dim, rot_dim;
    float eps;
    const void *in[3];  // q, k, v
    int64_t in_stride[3];
    const float *bias[3];
    const float *norm[2];
    const int32_t *positions;
    const float *inv_freq;
    void *q_out;
    int64_t q_out_stride;
    const int64_t *slots;  // with a pool
    void *k_dst, *v_dst;   // the pool's, or k_out and null
    int64_t k_row_stride;  // without a pool
    int64_t page_stride, token_stride, head_stride, n_pages;
    int shift;
};

template <int TYPE>
struct Elem;
template <>
struct Elem<MI355X_TYPE_F32> {
    typedef float T;
    __device__ static float up(T v) { return v; }
    __device__ static T down(float v) { return v; }
};
template <>
struct Elem<MI355X_TYPE_F16> {
    typedef _Float16 T;
    __device__ static float up(T v) { return static_cast<float>(v); }
    __device__ static T down(float v) { return static_cast<T>(v); }
};
template <>
struct Elem<MI355X_TYPE_BF16> {
    typedef __bf16 T;
    __device__ static float up(T v) { return static_cast<float>(v); }
    __device__ static T down(float v) { return static_cast<T>(v); }
};

__device__ __forceinline__ void turn(int32_t pos, float inv_freq, float *c, float *s) {
    const double rev = static_cast<double>(pos) * static_cast<double>(inv_freq) * 0.15915494309189533577;
    sincospif(2.0f * static_cast<float>(rev - rint(rev)), s, c);
}

__device__ __forceinline__ float group_sum(float v, int width) {
    for (int d = width >> 1; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Where head h (0 .. n_heads + 2 n_kv_heads) of a row goes; null: nowhere.
template <typename TO>
__device__ __forceinline__ TO *out_head(const RopeArgs &a, int64_t row, int which, int h) {
    if (which == 0) return static_cast<TO *>(a.q_out) + row * a.q_out_stride + static_cast<int64_t>(h) * a.head_dim;
    TO *base = static_cast<TO *>(which == 1 ? a.k_dst : a.v_dst);
    if (!a.slots) return base + row * a.k_row_stride + static_cast<int64_t>(h) * a.head_dim;
    const int64_t slot = a.slots[row];
    if (!slot_in_pool(slot, a.n_pages, a.shift)) return nullptr;
    return base + (slot >> a.shift) * a.page_stride + (slot & ((int64_t(1) << a.shift) - 1)) * a.token_stride +
           h * a.head_stride;
}

// Two runs of W values of a head per lane -- W pairs of the rotated part, or 2 W
// values behind it --, LANES lanes per head: head_dim and rot_dim are multiples
// of 2 W, and rows, strides and pages of 16 bytes.  A workgroup takes a row, forms
// its sines and cosines once, in LDS, and reads its input past the caches'
// replacement (read once).  8192 rows of 32 + 2 x 8 heads of 128, norms, 201 MB: 41
// us, 4.96 TB/s; 52 with W = 4 instead of 8 (16-byte loads of 16-bit values, where the
// sizes allow them), 48 with every lane's own sines, 45 with four rows to a
// workgroup, 44 with plain loads.
template <int TYPE, int W>
struct Run {
    typedef typename Elem<TYPE>::T V __attribute__((ext_vector_type(W)));
};

template <int IN, int OUT, bool PAIRS, int W, int LANES>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int heads, int rows_per_group) {
    typedef typename Elem<IN>::T TI;
    typedef typename Elem<OUT>::T TO;
    typedef typename Run<IN, W>::V VI;
    typedef typename Run<OUT, W>::V VO;
    typedef typename Run<MI355X_TYPE_F32, W>::V VF;
    constexpr int kHeadsAtOnce = 256 / LANES;
    const int u = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const int hd = a.head_dim, rot = a.rot_dim;
    const bool on = 2 * W * u < hd, turned = 2 * W * u < rot;
    // the lane's two runs
    const int i0 = !on ? 0 : turned && !PAIRS ? W * u : 2 * W * u;
    const int i1 = !on ? W : turned && !PAIRS ? rot / 2 + W * u : 2 * W * u + W;
    const int first_head = blockIdx.y * kHeadsAtOnce, step = gridDim.y * kHeadsAtOnce;
    __shared__ __attribute__((aligned(32))) float turns[2][256];  // cosines, sines; rot_dim <= 512
    const int64_t row_end = min(a.n_rows, (static_cast<int64_t>(blockIdx.x) + 1) * rows_per_group);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_group; row < row_end; ++row) {
        if (rot > 0) {
            const int32_t pos = a.positions[row];
            for (int p = threadIdx.x; p < rot / 2; p += 256) turn(pos, a.inv_freq[p], &turns[0][p], &turns[1][p]);
            __syncthreads();
        }
        VF c, s;
        if (turned) {
            c = *reinterpret_cast<const VF *>(&turns[0][W * u]);
            s = *reinterpret_cast<const VF *>(&turns[1][W * u]);
        }
        for (int hh = first_head + slot; hh < heads; hh += step) {
            const int which = hh < a.n_heads ? 0 : hh < a.n_heads + a.n_kv_heads ? 1 : 2;
            const int h = hh - (which == 0 ? 0 : which == 1 ? a.n_heads : a.n_heads + a.n_kv_heads);
            const TI *src = static_cast<const TI *>(which == 0 ? a.in[0] : which == 1 ? a.in[1] : a.in[2]) +
                            row * (which == 0 ? a.in_stride[0] : which == 1 ? a.in_stride[1] : a.in_stride[2]) +
                            static_cast<int64_t>(h) * hd;
            const float *bias = which == 0 ? a.bias[0] : which == 1 ? a.bias[1] : a.bias[2];
            const float *norm = which == 0 ? a.norm[0] : which == 1 ? a.norm[1] : nullptr;
            const int j0 = which == 2 ? 2 * W * u : i0, j1 = which == 2 ? 2 * W * u + W : i1;
            float x[2 * W];
            if (on) {
                const VI p = __builtin_nontemporal_load(reinterpret_cast<const VI *>(src + j0));
                const VI q = __builtin_nontemporal_load(reinterpret_cast<const VI *>(src + j1));
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    x[i] = Elem<IN>::up(p[i]);
                    x[W + i] = Elem<IN>::up(q[i]);
                }
                if (bias) {
                    const float *b = bias + static_cast<int64_t>(h) * hd;
                    const VF p1 = *reinterpret_cast<const VF *>(b + j0), q1 = *reinterpret_cast<const VF *>(b + j1);
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        x[i] += p1[i];
                        x[W + i] += q1[i];
                    }
                }
            }
            if (norm) {  // the same for all lanes of a head
                float ss = 0.0f;
                if (on)
#pragma unroll
                    for (int i = 0; i < 2 * W; ++i) ss = fmaf(x[i], x[i], ss);
                const float scale = 1.0f / sqrtf(group_sum(ss, LANES) / static_cast<float>(hd) + a.eps);
                if (on) {
                    const VF p1 = *reinterpret_cast<const VF *>(norm + j0), q1 = *reinterpret_cast<const VF *>(norm + j1);
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        x[i] = x[i] * scale * p1[i];
                        x[W + i] = x[W + i] * scale * q1[i];
                    }
                }
            }
            if (turned && which != 2) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int m = PAIRS ? 2 * i : i, n = PAIRS ? 2 * i + 1 : W + i;
                    const float v = x[m], w = x[n];
                    x[m] = v * c[i] - w * s[i];
                    x[n] = w * c[i] + v * s[i];
                }
            }
            TO *dst = on ? out_head<TO>(a, row, which, h) : nullptr;
            if (dst) {
                VO p, q;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    p[i] = Elem<OUT>::down(x[i]);
                    q[i] = Elem<OUT>::down(x[W + i]);
                }
                *reinterpret_cast<VO *>(dst + j0) = p;
                *reinterpret_cast<VO *>(dst + j1) = q;
            }
        }
        if (rot > 0 && row + 1 < row_end) __syncthreads();
    }
}

// Any sizes and alignments: one wavefront per row and head, value by value.
template <int IN, int OUT, bool PAIRS>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs a, int heads, int64_t items) {
    typedef typename Elem<IN>::T TI;
    typedef typename Elem<OUT>::T TO;
    const int lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= items) return;
    const int64_t row = item / heads;
    const int hh = static_cast<int>(item % heads);
    const int which = hh < a.n_heads ? 0 : hh < a.n_heads + a.n_kv_heads ? 1 : 2;
    const int h = hh - (which == 0 ? 0 : which == 1 ? a.n_heads : a.n_heads + a.n_kv_heads);
    const int hd = a.head_dim, rot = which == 2 ? 0 : a.rot_dim;
    TO *dst = out_head<TO>(a, row, which, h);
    if (!dst) return;
    const TI *src = static_cast<const TI *>(a.in[which]) + row * a.in_stride[which] + static_cast<int64_t>(h) * hd;
    const float *bias = a.bias[which] ? a.bias[which] + static_cast<int64_t>(h) * hd : nullptr;
    const float *norm = which < 2 ? a.norm[which] : nullptr;
    auto value = [&](int i) { return Elem<IN>::up(src[i]) + (bias ? bias[i] : 0.0f); };
    float scale = 1.0f;
    if (norm) {
        float ss = 0.0f;
        for (int i = lane; i < hd; i += 64) {
            const float v = value(i);
            ss = fmaf(v, v, ss);
        }
        scale = 1.0f / sqrtf(group_sum(ss, 64) / static_cast<float>(hd) + a.eps);
    }
    auto normed = [&](int i) { return norm ? value(i) * scale * norm[i] : value(i); };
    for (int p = lane; p < rot / 2; p += 64) {
        const int i = PAIRS ? 2 * p : p, j = PAIRS ? 2 * p + 1 : p + rot / 2;
        const float x = normed(i), y = normed(j);
        float c, s;
        turn(a.positions[row], a.inv_freq[p], &c, &s);
        dst[i] = Elem<OUT>::down(x * c - y * s);
        dst[j] = Elem<OUT>::down(y * c + x * s);
    }
    for (int i = rot + lane; i < hd; i += 64) dst[i] = Elem<OUT>::down(normed(i));
}

template <int IN, int OUT, bool PAIRS, int W, int LANES>
int launch_rope_lanes(mi355x_ctx *ctx, const RopeArgs &a) {
    const int heads = a.n_heads + (a.slots ? 2 : 1) * a.n_kv_heads;
    const int64_t at_once = 256 / LANES, passes = (heads + at_once - 1) / at_once;
    // few rows: a workgroup per row and pass over its heads (one row of 20 heads of 128:
    // 3.9 us against 4.1); many: one per row
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>(passes, 4 * ctx->num_cus / std::max<int64_t>(1, a.n_rows)));
    constexpr int64_t kMostGroups = int64_t(1) << 22;
    const int rows_per_group = static_cast<int>((a.n_rows + kMostGroups - 1) / kMostGroups);
    const dim3 grid(static_cast<unsigned>((a.n_rows + rows_per_group - 1) / rows_per_group), static_cast<unsigned>(split));
    rope_kernel<IN, OUT, PAIRS, W, LANES><<<grid, 256, 0, ctx->stream>>>(a, heads, rows_per_group);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

template <int IN, int OUT, bool PAIRS>
int launch_rope_any(mi355x_ctx *ctx, const RopeArgs &a) {
    const int heads = a.n_heads + (a.slots ? 2 : 1) * a.n_kv_heads;
    constexpr int64_t kMostItems = int64_t(1) << 25;  // wavefronts of a launch
    for (int64_t row = 0; row < a.n_rows;) {
        const int64_t rows = std::min(a.n_rows - row, std::max<int64_t>(1, kMostItems / heads));
        RopeArgs b = a;
        for (int i = 0; i < 3; ++i)
            if (b.in[i]) b.in[i] = static_cast<const typename Elem<IN>::T *>(a.in[i]) + row * a.in_stride[i];
        b.q_out = static_cast<typename Elem<OUT>::T *>(a.q_out) + row * a.q_out_stride;
        if (a.positions) b.positions = a.positions + row;
        if (a.slots) b.slots = a.slots + row;
        else b.k_dst = static_cast<typename Elem<OUT>::T *>(a.k_dst) + row * a.k_row_stride;
        rope_any_kernel<IN, OUT, PAIRS>
            <<<static_cast<unsigned>((rows * heads + 3) / 4), 256, 0, ctx->stream>>>(b, heads, rows * heads);
        MI355X_HIP(hipGetLastError());
        row += rows;
    }
    return MI355X_OK;
}

bool whole_chunks(const void *p, int64_t stride, int64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * bytes % 16 == 0;
}

template <int IN, int OUT, bool PAIRS>
int launch_rope_pairs(mi355x_ctx *ctx, const RopeArgs &a) {
    constexpr int64_t ib = sizeof(typename Elem<IN>::T), ob = sizeof(typename Elem<OUT>::T);
    bool fast = a.head_dim % 8 == 0 && a.rot_dim % 8 == 0 && a.head_dim <= 512 &&
                whole_chunks(a.q_out, a.q_out_stride, ob) && whole_chunks(a.inv_freq, 0, 4);
    for (int i = 0; i < 3; ++i) fast = fast && whole_chunks(a.in[i], a.in_stride[i], ib) && whole_chunks(a.bias[i], 0, 4);
    for (int i = 0; i < 2; ++i) fast = fast && whole_chunks(a.norm[i], 0, 4);
    if (!a.slots) fast = fast && whole_chunks(a.k_dst, a.k_row_stride, ob);
    if (!fast) return launch_rope_any<IN, OUT, PAIRS>(ctx, a);
    if (a.head_dim % 16 == 0 && a.rot_dim % 16 == 0) {
        if (a.head_dim <= 64) return launch_rope_lanes<IN, OUT, PAIRS, 8, 4>(ctx, a);
        if (a.head_dim <= 128) return launch_rope_lanes<IN, OUT, PAIRS, 8, 8>(ctx, a);
        if (a.head_dim <= 256) return launch_rope_lanes<IN, OUT, PAIRS, 8, 16>(ctx, a);
        return launch_rope_lanes<IN, OUT, PAIRS, 8, 32>(ctx, a);
    }
    if (a.head_dim <= 64) return launch_rope_lanes<IN, OUT, PAIRS, 4, 8>(ctx, a);
    if (a.head_dim <= 128) return launch_rope_lanes<IN, OUT, PAIRS, 4, 16>(ctx, a);
    if (a.head_dim <= 256) return launch_rope_lanes<IN, OUT, PAIRS, 4, 32>(ctx, a);
    return launch_rope_lanes<IN, OUT, PAIRS, 4, 64>(ctx, a);
}

template <int IN, int OUT>
int launch_rope(mi355x_ctx *ctx, const RopeArgs &a, bool pairs) {
    return pairs ? launch_rope_pairs<IN, OUT, true>(ctx, a) : launch_rope_pairs<IN, OUT, false>(ctx, a);
}

template <int OUT>
int launch_rope_in(mi355x_ctx *ctx, const RopeArgs &a, int in_type, bool pairs) {
    switch (in_type) {
    case MI355X_TYPE_F32: return launch_rope<MI355X_TYPE_F32, OUT>(ctx, a, pairs);
    case MI355X_TYPE_F16: return launch_rope<MI355X_TYPE_F16, OUT>(ctx, a, pairs);
    default: return launch_rope<MI355X_TYPE_BF16, OUT>(ctx, a, pairs);
    }
}

}  // namespace

int launch_qk_norm_rope(mi355x_ctx *ctx, const mi355x_qk_norm_rope_args &u) {
    RopeArgs a{};
    a.n_rows = u.n_rows;
    a.n_heads = u.n_heads;
    a.n_kv_heads = u.n_kv_heads;
    a.head_dim = u.head_dim;
    a.rot_dim = u.rot_dim;
    a.eps = u.eps;
    const void *in[3] = {u.q, u.k, u.pool ? u.v : nullptr};
    const int64_t st[3] = {u.q_stride, u.k_stride, u.v_stride};
    const float *bias[3] = {u.q_bias, u.k_bias, u.v_bias};
    for (int i = 0; i < 3; ++i) {
        a.in[i] = in[i];
        a.in_stride[i] = st[i];
        a.bias[i] = bias[i];
    }
    a.norm[0] = u.q_norm;
    a.norm[1] = u.k_norm;
    a.positions = u.positions;
    a.inv_freq = u.inv_freq;
    a.q_out = u.q_out;
    a.q_out_stride = u.q_out_stride;
    if (u.pool) {
        a.slots = u.slots;
        a.k_dst = u.pool->k;
        a.v_dst = u.pool->v;
        a.page_stride = u.pool->page_stride;
        a.token_stride = u.pool->token_stride;
        a.head_stride = u.pool->head_stride;
        a.n_pages = u.pool->n_pages;
        a.shift = __builtin_ctz(static_cast<unsigned>(u.pool->page_tokens));
    } else {
        a.k_dst = u.k_out;
        a.k_row_stride = u.k_out_stride;
    }
    const bool pairs = u.rope_mode == MI355X_ROPE_PAIRS;
    switch (u.out_type) {
    case MI355X_TYPE_F32: return launch_rope_in<MI355X_TYPE_F32>(ctx, a, u.in_type, pairs);
    case MI355X_TYPE_F16: return launch_rope_in<MI355X_TYPE_F16>(ctx, a, u.in_type, pairs);
    default: return launch_rope_in<MI355X_TYPE_BF16>(ctx, a, u.in_type, pairs);
    }
}

}  // namespace mi355x
