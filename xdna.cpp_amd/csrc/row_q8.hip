// Rows in 8 bits: the residual's addition with the root-mean-square norm, and
// the gated product, each with the largest magnitude of the row as its scale.
//
// Codes are rint(t * 127 / max |t|) in 64-bit arithmetic: the values t are formed
// there (a product of two f32 numbers is exact in it), a multiplication by 127 /
// max |t| gives the code, and one that lands near to a border is settled by the
// division itself.  The norm's root multiplies a whole row, so it meets the scale
// alone.
#include "internal.h"
#include "row_values.h"

#include <algorithm>
#include <type_traits>

namespace mi355x {
namespace {

constexpr int kMostWaves = 16;

struct RowArgs {
    int64_t n_rows;
    int n;
    int type, residual_type;
    const void *x, *y;  // norm: x and the residual; gate and up
    int64_t x_stride, y_stride;
    void *y_out;
    int64_t y_out_stride;
    const float *norm;
    float eps;
    int8_t *q;
    int64_t q_stride;
    float *scales;
};

// The code of t in a row whose largest magnitude is `most` > 0; unit = 127 / most.
// t * unit is within 2^-44 of the stated quotient.
__device__ __forceinline__ int code_of(double t, double most, double unit) {
    const double y = t * unit, r = rint(y);
    if (fabs(y - r) < 0.5 - 1e-9) return static_cast<int>(r);
    return static_cast<int>(rint(t * 127.0 / most));
}

// Sum and largest over the workgroup's threads, one after the other in `lds`.
__device__ __forceinline__ void group_sum_max(double *sum, double *most, double (*lds)[2]) {
    const int wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
    const double s = wave_sum64(*sum), m = wave_max64(*most);
    if ((threadIdx.x & 63) == 0) {
        lds[wave][0] = s;
        lds[wave][1] = m;
    }
    __syncthreads();
    double ts = 0.0, tm = 0.0;
    for (int w = 0; w < waves; ++w) {
        ts += lds[w][0];
        tm = fmax(tm, lds[w][1]);
    }
    *sum = ts;
    *most = tm;
}

template <class F>
__device__ __forceinline__ void by_type(int type, F f) {
    if (type == MI355X_TYPE_F32) f(std::integral_constant<int, MI355X_TYPE_F32>{});
    else if (type == MI355X_TYPE_F16) f(std::integral_constant<int, MI355X_TYPE_F16>{});
    else f(std::integral_constant<int, MI355X_TYPE_BF16>{});
}

__device__ __forceinline__ void load_as_float(const void *row, int type, int i, int n, float *v) {
    by_type(type, [&](auto t) {
        const auto r = row_load8<decltype(t)::value>(row, i, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(r[j]);
    });
}

__device__ __forceinline__ const void *row_at(const void *p, int type, int64_t values) {
    return static_cast<const uint8_t *>(p) + values * (type == MI355X_TYPE_F32 ? 4 : 2);
}

// The eight values t of a norm's row, and the squares of h.  First pass: h is
// formed and stored; second: read where it was stored.
__device__ __forceinline__ void norm_values(const RowArgs &a, int64_t row, int i, bool second, double *t,
                                            double *squares) {
    float h[8];
    if (second && a.y_out) {
        load_as_float(row_at(a.y_out, a.residual_type, row * a.y_out_stride), a.residual_type, i, a.n, h);
    } else {
        load_as_float(row_at(a.x, a.type, row * a.x_stride), a.type, i, a.n, h);
        if (a.y) {
            by_type(a.residual_type, [&](auto ty) {
                constexpr int TYPE = decltype(ty)::value;
                typedef typename RowElem<TYPE>::T T;
                auto r = row_load8<TYPE>(row_at(a.y, TYPE, row * a.y_stride), i, a.n);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    r[j] = static_cast<T>(h[j] + static_cast<float>(r[j]));
                    h[j] = static_cast<float>(r[j]);
                }
                if (a.y_out)
                    row_store8<TYPE>(const_cast<void *>(row_at(a.y_out, TYPE, row * a.y_out_stride)), i, a.n, r);
            });
        }
    }
    float w[8];
    if (a.norm) load_as_float(a.norm, MI355X_TYPE_F32, i, a.n, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double d = h[j];
        *squares = fma(d, d, *squares);
        t[j] = a.norm ? d * static_cast<double>(w[j]) : d;
    }
}

__device__ __forceinline__ void swiglu_values(const RowArgs &a, int64_t row, int i, double *t) {
    float g[8], u[8];
    load_as_float(row_at(a.x, a.type, row * a.x_stride), a.type, i, a.n, g);
    load_as_float(row_at(a.y, a.type, row * a.y_stride), a.type, i, a.n, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double d = g[j];
        t[j] = d / (1.0 + exp(-d)) * static_cast<double>(u[j]);
    }
}

// A workgroup per row, the row's values formed twice: for the largest, and for
// the codes.
template <bool GATED>
__global__ __launch_bounds__(64 * kMostWaves) void row_q8_kernel(RowArgs a) {
    __shared__ double lds[2][kMostWaves][2];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x, turn ^= 1) {
        double sum = 0.0, most = 0.0;
        for (int i = 8 * threadIdx.x; i < a.n; i += 8 * blockDim.x) {
            double t[8];
            if (GATED) swiglu_values(a, row, i, t);
            else norm_values(a, row, i, false, t, &sum);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                most = fmax(most, fabs(t[j]));
                sum = fma(t[j], 0.0, sum);  // NaN where t is not finite
            }
        }
        group_sum_max(&sum, &most, lds[turn]);
        const bool bad = !(fabs(sum) <= 1.7976931348623157e308);
        const bool zero = bad || most == 0.0;
        const double unit = zero ? 0.0 : 127.0 / most;
        if (threadIdx.x == 0) {
            double scale = most / 127.0;
            if (!GATED && a.norm) scale = most / sqrt(sum / a.n + static_cast<double>(a.eps)) / 127.0;
            if (most == 0.0) scale = 0.0;
            a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(scale);
        }
        for (int i = 8 * threadIdx.x; i < a.n; i += 8 * blockDim.x) {
            double t[8], ignored = 0.0;
            if (GATED) swiglu_values(a, row, i, t);
            else norm_values(a, row, i, true, t, &ignored);
            uint32_t c[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!zero) c[j >> 2] |= (static_cast<uint32_t>(code_of(t[j], most, unit)) & 255u) << (8 * (j & 3));
            row_store_codes(a.q + row * a.q_stride, i, a.n, c[0], c[1]);
        }
    }
}

template <bool GATED>
int launch_rows(mi355x_ctx *ctx, const RowArgs &a) {
    const int threads = std::min(64 * kMostWaves, (a.n + 511) / 512 * 64);
    const int64_t groups = std::min<int64_t>(a.n_rows, 1 << 20);
    row_q8_kernel<GATED><<<static_cast<unsigned>(groups), threads, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace

int launch_norm_q8(mi355x_ctx *ctx, const mi355x_norm_q8_args &u) {
    RowArgs a{};
    a.n_rows = u.n_rows;
    a.n = u.n;
    a.type = u.type;
    a.x = u.x;
    a.x_stride = u.x_stride;
    a.residual_type = u.residual_type;
    a.y = u.residual;
    a.y_stride = u.residual_stride;
    a.y_out = u.residual_out;
    a.y_out_stride = u.residual_out_stride;
    a.norm = u.norm;
    a.eps = u.eps;
    a.q = u.q;
    a.q_stride = u.q_stride;
    a.scales = u.scales;
    return launch_rows<false>(ctx, a);
}

int launch_swiglu_q8(mi355x_ctx *ctx, const mi355x_swiglu_q8_args &u) {
    RowArgs a{};
    a.n_rows = u.n_rows;
    a.n = u.n;
    a.type = u.type;
    a.x = u.gate;
    a.x_stride = u.gate_stride;
    a.y = u.up;
    a.y_stride = u.up_stride;
    a.q = u.q;
    a.q_stride = u.q_stride;
    a.scales = u.scales;
    return launch_rows<true>(ctx, a);
}

}  // namespace mi355x
