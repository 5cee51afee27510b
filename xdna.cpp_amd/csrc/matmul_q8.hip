// Products of 8-bit integers with a scale for each row and each channel, on the
// integer matrix cores: sums of products of codes are exact in 32 bits (128 * 128
// * 131056 < 2^31), so the order of the sum and the split of the work do not show.
#include "internal.h"
#include "device_common.h"

#include <algorithm>

namespace mi355x {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct MatmulArgs {
    int64_t x_stride, w_stride, out_stride;
    const int8_t *x, *w;
    const float *x_scales, *w_scales, *bias;
    void *out;
    int m, n, k, out_type;
};

// One value of the product, in the stated order of roundings.
__device__ __forceinline__ float scaled(int sum, float ws, float xs, bool has_bias, float bias) {
#pragma clang fp contract(off)
    float v = static_cast<float>(sum) * ws;
    v = v * xs;
    if (has_bias) v = v + bias;
    return v;
}

__device__ __forceinline__ void store_value(const MatmulArgs &a, int64_t at, float v) {
    if (a.out_type == MI355X_TYPE_F32) static_cast<float *>(a.out)[at] = v;
    else if (a.out_type == MI355X_TYPE_F16) static_cast<_Float16 *>(a.out)[at] = static_cast<_Float16>(v);
    else static_cast<__bf16 *>(a.out)[at] = static_cast<__bf16>(v);
}

// A wavefront per 16 rows and 16 channels.
__global__ __launch_bounds__(256) void matmul_q8_kernel(MatmulArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int blocks = (a.n + 63) / 64;
    const int m0 = blockIdx.x / blocks * 16, n0 = blockIdx.x % blocks * 64 + 16 * wave;
    if (n0 >= a.n) return;
    const int8_t *w = a.w + static_cast<int64_t>(min(n0 + col, a.n - 1)) * a.w_stride + 16 * quad;
    const int8_t *x = a.x + static_cast<int64_t>(min(m0 + col, a.m - 1)) * a.x_stride + 16 * quad;
    i32x4 c = {0, 0, 0, 0};
    for (int k = 0; k < a.k; k += 64) {
        i32x4 wf = {0, 0, 0, 0}, xf = {0, 0, 0, 0};
        if (k + 16 * quad < a.k) {
            wf = *reinterpret_cast<const i32x4 *>(w + k);
            xf = *reinterpret_cast<const i32x4 *>(x + k);
        }
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, c, 0, 0, 0);
    }
    const int m = m0 + col;
    if (m >= a.m) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + 4 * quad + i;
        if (n < a.n)
            store_value(a, m * a.out_stride + n,
                        scaled(c[i], a.w_scales[n], a.x_scales[m], a.bias != nullptr, a.bias ? a.bias[n] : 0.0f));
    }
}

}  // namespace

size_t matmul_q8_workspace_bytes(const mi355x_ctx *ctx) { return static_cast<size_t>(ctx->num_cus) * 65536 + 65536; }

int launch_matmul_q8(mi355x_ctx *ctx, const mi355x_matmul_q8_args &u) {
    MatmulArgs a{};
    a.x_stride = u.x_stride;
    a.w_stride = u.w_stride;
    a.out_stride = u.out_stride;
    a.x = u.x;
    a.w = u.w;
    a.x_scales = u.x_scales;
    a.w_scales = u.w_scales;
    a.bias = u.bias;
    a.out = u.out;
    a.m = static_cast<int>(u.n_rows);
    a.n = static_cast<int>(u.n_out);
    a.k = static_cast<int>(u.k);
    a.out_type = u.out_type;
    const int64_t groups = (u.n_rows + 15) / 16 * ((u.n_out + 63) / 64);
    if (groups >= (1 << 23))
        return set_error(MI355X_EUNSUPPORTED, "mi355x_matmul_q8: " + std::to_string(groups) + " blocks, 2^23 or more");
    matmul_q8_kernel<<<static_cast<unsigned>(groups), 256, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace mi355x
