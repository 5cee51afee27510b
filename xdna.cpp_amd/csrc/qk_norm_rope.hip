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

template <int IN, int OUT>
int launch_rope(mi355x_ctx *ctx, const RopeArgs &a, bool pairs) {
    const int heads = a.n_heads + (a.slots ? 2 : 1) * a.n_kv_heads;
    const int64_t items = a.n_rows * heads;
    // HIP takes up to 2^32 - 1 threads of a launch in x
    constexpr int64_t kMostItems = int64_t(1) << 25;
    for (int64_t row = 0; row < a.n_rows;) {
        const int64_t rows = std::min(a.n_rows - row, std::max<int64_t>(1, kMostItems / heads));
        RopeArgs b = a;
        b.n_rows = rows;
        for (int i = 0; i < 3; ++i)
            if (b.in[i]) b.in[i] = static_cast<const typename Elem<IN>::T *>(a.in[i]) + row * a.in_stride[i];
        b.q_out = static_cast<typename Elem<OUT>::T *>(a.q_out) + row * a.q_out_stride;
        if (a.positions) b.positions = a.positions + row;
        if (a.slots) b.slots = a.slots + row;
        else b.k_dst = static_cast<typename Elem<OUT>::T *>(a.k_dst) + row * a.k_row_stride;
        const unsigned grid = static_cast<unsigned>((rows * heads + 3) / 4);
        if (pairs) rope_any_kernel<IN, OUT, true><<<grid, 256, 0, ctx->stream>>>(b, heads, rows * heads);
        else rope_any_kernel<IN, OUT, false><<<grid, 256, 0, ctx->stream>>>(b, heads, rows * heads);
        MI355X_HIP(hipGetLastError());
        row += rows;
    }
    (void)items;
    return MI355X_OK;
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
