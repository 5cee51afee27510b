// Attention of new tokens over a paged KV cache.
//
// One pass over a row's keys with the running maximum m and sum l of the
// softmax: a key's score s moves m to max(m, s), scales what was summed by
// exp(m_old - m), and adds exp(s - m) v and exp(s - m).
#include "internal.h"
#include "paged_index.h"

#include <algorithm>

namespace mi355x {
namespace {

template <int TYPE>
struct Half;
template <>
struct Half<MI355X_TYPE_F16> {
    typedef _Float16 T;
};
template <>
struct Half<MI355X_TYPE_BF16> {
    typedef __bf16 T;
};

__device__ __forceinline__ float wave_total(float v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// One wavefront per row and head, key by key; a lane holds values lane + 64 i.
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void attention_rows_kernel(mi355x_paged_attention_args a, mi355x_kv_pool pool,
                                                             int shift) {
    typedef typename Half<TYPE>::T T;
    constexpr int kPer = (HD + 63) / 64;
    const int lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int64_t row = item / a.n_heads;
    const int h = static_cast<int>(item % a.n_heads);
    if (row >= a.n_rows) return;
    const int s = seq_of_row(a.row_offsets, a.n_seqs, row);
    if (s < 0) return;
    const int64_t kv = a.kv_lens[s], pos = kv - (a.row_offsets[s + 1] - row);
    const KeyRange keys =
        visible_keys(pos, kv, static_cast<int64_t>(a.table_cols) << shift, a.window, a.causal != 0);
    const int kvh = h / (a.n_heads / pool.n_kv_heads);
    const int32_t *table = a.block_table + s * a.table_stride;
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + static_cast<int64_t>(h) * HD;
    float qf[kPer], o[kPer];
    for (int i = 0; i < kPer; ++i) {
        qf[i] = lane + 64 * i < HD ? static_cast<float>(q[lane + 64 * i]) : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = keys.lo; j < keys.hi; ++j) {
        const int32_t page = table[j >> shift];
        if (!page_in_pool(page, pool.n_pages)) continue;
        const int64_t at = page * pool.page_stride + (j & ((int64_t(1) << shift) - 1)) * pool.token_stride +
                           kvh * pool.head_stride;
        const T *k = static_cast<const T *>(pool.k) + at, *v = static_cast<const T *>(pool.v) + at;
        float dot = 0.0f;
        for (int i = 0; i < kPer; ++i)
            if (lane + 64 * i < HD) dot = fmaf(qf[i], static_cast<float>(k[lane + 64 * i]), dot);
        float sc = wave_total(dot) * a.scale;
        if (a.softcap > 0.0f) sc = a.softcap * tanhf(sc / a.softcap);
        const float m_new = fmaxf(m, sc), base = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = expf(m - base), p = expf(sc - base);
        l = l * keep + p;
        for (int i = 0; i < kPer; ++i) {
            const float vi = lane + 64 * i < HD ? static_cast<float>(v[lane + 64 * i]) : 0.0f;
            o[i] = o[i] * keep + (p == 0.0f ? 0.0f : p * vi);
        }
        m = m_new;
    }
    const int64_t at = row * a.out_stride + static_cast<int64_t>(h) * HD;
    for (int i = 0; i < kPer; ++i) {
        if (lane + 64 * i >= HD) continue;
        const float v = l == 0.0f ? 0.0f : o[i] / l;
        if (a.out_type == MI355X_TYPE_F32) static_cast<float *>(a.out)[at + lane + 64 * i] = v;
        else static_cast<T *>(a.out)[at + lane + 64 * i] = static_cast<T>(v);
    }
}

template <int TYPE>
int launch_rows(mi355x_ctx *ctx, const mi355x_paged_attention_args &a, int shift) {
    const dim3 grid(static_cast<unsigned>((a.n_rows * a.n_heads + 3) / 4));
    switch (a.pool->head_dim) {
    case 64: attention_rows_kernel<TYPE, 64><<<grid, 256, 0, ctx->stream>>>(a, *a.pool, shift); break;
    case 96: attention_rows_kernel<TYPE, 96><<<grid, 256, 0, ctx->stream>>>(a, *a.pool, shift); break;
    case 128: attention_rows_kernel<TYPE, 128><<<grid, 256, 0, ctx->stream>>>(a, *a.pool, shift); break;
    default: attention_rows_kernel<TYPE, 256><<<grid, 256, 0, ctx->stream>>>(a, *a.pool, shift); break;
    }
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace

size_t paged_attention_workspace_bytes(const mi355x_ctx *, int, int, int) { return 256; }

int launch_paged_attention(mi355x_ctx *ctx, const mi355x_paged_attention_args &a) {
    const int shift = __builtin_ctz(static_cast<unsigned>(a.pool->page_tokens));
    return a.pool->type == MI355X_TYPE_F16 ? launch_rows<MI355X_TYPE_F16>(ctx, a, shift)
                                           : launch_rows<MI355X_TYPE_BF16>(ctx, a, shift);
}

}  // namespace mi355x
