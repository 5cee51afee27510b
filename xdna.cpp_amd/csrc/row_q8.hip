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

__device__ __forceinline__ double gated(float g, float u) {
    const double d = g;
    return d / (1.0 + exp(-d)) * static_cast<double>(u);
}
// For single values: a function of its own, so that the exponential's numbers do not take up
// the registers of a kernel's values (4096 gated rows of 14336: 90 us with them).
__device__ __attribute__((noinline)) double gated_value(float g, float u) { return gated(g, u); }

__device__ __forceinline__ void swiglu_values(const RowArgs &a, int64_t row, int i, double *t) {
    float g[8], u[8];
    load_as_float(row_at(a.x, a.type, row * a.x_stride), a.type, i, a.n, g);
    load_as_float(row_at(a.y, a.type, row * a.y_stride), a.type, i, a.n, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = gated(g[j], u[j]);
}

// Rows longer than a workgroup's registers: the values formed twice, for the largest
// and for the codes.
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
            row_store_codes(a.q + row * a.q_stride, i, a.n, static_cast<uint64_t>(c[1]) << 32 | c[0]);
        }
    }
}

// ---- rows held in registers ------------------------------------------------------

// One pass: a row is read once, its sum of squares and its largest magnitude meet in one
// reduction over the workgroup, and codes leave from registers.  Bound by memory: the norm
// of 8192 rows of 8192 in bf16 with its residual, 470 MB, takes 91 us (5.2 TB/s, as a copy);
// gates of 4096 x 14336 in bf16, 294 MB, 63 us (4.7 TB/s; besides memory some 20 vector
// operations and two of a quarter's rate a value; rows of zeros, and others that f32 will not
// do for, are formed in 64 bits: 191).  One row: what a launch takes, 4 and 5 us.
// A thread has CHUNKS runs of 8 values, so rows of up to 8 * CHUNKS * threads values
// are read once.
constexpr int kMostChunks = 4;
constexpr int kMostHeld = 8 * kMostChunks * 64 * kMostWaves;

// Whether all threads' runs number c lie in the row, which the whole workgroup asks at once.
__device__ __forceinline__ bool all_in(int c, int n) { return 8 * (c + 1) * static_cast<int>(blockDim.x) <= n; }

template <int TYPE, int CHUNKS>
__device__ __forceinline__ void load_row(const void *p, int n, typename RowElem<TYPE>::Raw8 *r) {
    const int first = 8 * threadIdx.x, step = 8 * blockDim.x;
    if (CHUNKS == 1) {
        r[0] = row_load8<TYPE>(p, first, n);
        return;
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) r[c] = row_load8_near<TYPE>(p, first + c * step, n);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (!all_in(c, n)) row_end<TYPE>(r[c], first + c * step, n);
}

// Codes, a byte each, of t * unit with `unit` next to 127 / most: 1.5 * 2^23 is added in
// the multiplication's own rounding, which leaves the nearest whole number in the low
// bits.  A bit of *doubt is set for each product nearer than error + slope |t| to a border.
template <bool SLOPE>
__device__ __forceinline__ uint64_t pack_codes(const float *t, float unit, float error, float slope, uint32_t *doubt) {
    constexpr float kWhole = 12582912.0f;
    float z[8], worst = 0.0f;
    auto off = [&](int j) {
        const float d = fabsf(fmaf(t[j], unit, kWhole - z[j]));
        return SLOPE ? fmaf(fabsf(t[j]), slope, d) : d;
    };
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        z[j] = fmaf(t[j], unit, kWhole);
        worst = fmaxf(worst, off(j));
    }
    uint32_t c[2];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        auto bits = [&](int j) { return __builtin_bit_cast(uint32_t, z[4 * d + j]); };
        // the low bytes of two, and of two such pairs
        const uint32_t lo = __builtin_amdgcn_perm(bits(1), bits(0), 0x0C0C0400u);
        const uint32_t hi = __builtin_amdgcn_perm(bits(3), bits(2), 0x0C0C0400u);
        c[d] = lo | hi << 16;
    }
    *doubt = 0;
    if (worst >= 0.5f - error)
#pragma unroll
        for (int j = 0; j < 8; ++j) *doubt |= off(j) >= 0.5f - error ? 1u << j : 0u;
    return c[0] | static_cast<uint64_t>(c[1]) << 32;
}

// The codes with those in doubt from exact(j).
template <class F>
__device__ __forceinline__ uint64_t settle_codes(uint64_t codes, uint32_t doubt, F exact) {
    while (doubt) {
        const int j = __builtin_ctz(doubt);
        doubt &= doubt - 1;
        const uint64_t code = static_cast<uint64_t>(exact(j) & 255) << (8 * j);
        codes = (codes & ~(uint64_t(255) << (8 * j))) | code;
    }
    return codes;
}

// Value i of a row, read again.
__device__ __forceinline__ float value_at(const void *p, int type, int64_t i) {
    if (type == MI355X_TYPE_F32) return static_cast<const float *>(p)[i];
    if (type == MI355X_TYPE_F16) return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
    return static_cast<float>(static_cast<const __bf16 *>(p)[i]);
}

// Largest magnitudes that leave f32's range neither way when 127 is divided by them.
__device__ __forceinline__ bool in_range(double most) { return most > 0x1p-60 && most < 0x1p100; }

template <int XT, int RT, int CHUNKS>
__global__ __launch_bounds__(64 * kMostWaves) void norm_rows_kernel(RowArgs a) {
    constexpr bool kResidual = RT >= 0;
    constexpr int kRes = kResidual ? RT : MI355X_TYPE_F32;
    typedef typename RowElem<kRes>::T ResT;
    __shared__ double lds[2][kMostWaves][2];
    const int first = 8 * threadIdx.x, step = 8 * blockDim.x;
    typename RowElem<MI355X_TYPE_F32>::Raw8 w[CHUNKS];
    if (a.norm) {
        load_row<MI355X_TYPE_F32, CHUNKS>(a.norm, a.n, w);
    } else {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[c][j] = 1.0f;
    }
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x, turn ^= 1) {
        float h[CHUNKS][8];
        {
            typename RowElem<XT>::Raw8 x[CHUNKS];
            typename RowElem<kRes>::Raw8 r[CHUNKS];
            load_row<XT, CHUNKS>(row_at(a.x, XT, row * a.x_stride), a.n, x);
            if (kResidual) load_row<kRes, CHUNKS>(row_at(a.y, kRes, row * a.y_stride), a.n, r);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    h[c][j] = static_cast<float>(x[c][j]);
                    if (kResidual) {
                        r[c][j] = static_cast<ResT>(h[c][j] + static_cast<float>(r[c][j]));
                        h[c][j] = static_cast<float>(r[c][j]);
                    }
                }
                if (kResidual && a.y_out)
                    row_store8<kRes>(const_cast<void *>(row_at(a.y_out, kRes, row * a.y_out_stride)), first + c * step,
                                     a.n, r[c]);
            }
        }
        double sum = 0.0, most = 0.0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double d = h[c][j], t = d * static_cast<double>(w[c][j]);
                sum = fma(d, d, sum);
                sum = fma(t, 0.0, sum);  // NaN where t is not finite
                most = fmax(most, fabs(t));
            }
        group_sum_max(&sum, &most, lds[turn]);
        const bool bad = !(fabs(sum) <= 1.7976931348623157e308), zero = bad || most == 0.0;
        const double unit = zero ? 0.0 : 127.0 / most;
        if (threadIdx.x == 0) {
            double scale = most / 127.0;
            if (a.norm) scale = most / sqrt(sum / a.n + static_cast<double>(a.eps)) / 127.0;
            a.scales[row] = bad ? __builtin_nanf("") : most == 0.0 ? 0.0f : static_cast<float>(scale);
        }
        int8_t *q = a.q + row * a.q_stride;
        // h w and the unit are off by half a step each, 2^-23 of 127 together; outside f32's
        // range every code is formed in 64 bits
        const bool near = in_range(most);
        const float unit32 = near && !bad ? static_cast<float>(unit) : 0.0f, error = near || zero ? 5e-5f : 1.0f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int i = first + c * step;
            if (i >= a.n) break;
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = near && !bad ? h[c][j] * w[c][j] : 0.0f;
            uint32_t doubt;
            uint64_t codes = pack_codes<false>(t, unit32, error, 0.0f, &doubt);
            codes = settle_codes(codes, doubt, [&](int j) {
                if (i + j >= a.n) return 0;
                float again;
                if (kResidual && a.y_out) {
                    again = value_at(a.y_out, kRes, row * a.y_out_stride + i + j);
                } else {
                    again = value_at(a.x, XT, row * a.x_stride + i + j);
                    if (kResidual)
                        again = static_cast<float>(static_cast<ResT>(again + value_at(a.y, kRes, row * a.y_stride + i + j)));
                }
                const double t = static_cast<double>(again) * (a.norm ? static_cast<double>(a.norm[i + j]) : 1.0);
                return code_of(t, most, unit);
            });
            row_store_codes(q, i, a.n, codes);
        }
    }
}

// The same in f32.  In units of 2^-24, 2^it is off by 1.22 |g| (the exponent -g log2 e and
// its constant) and 2, which for g > 0 the sum with 1 makes less of; the sum, its inverse
// and two products add 5: 17 units of t where g >= -8.  Below, 0.05 units of u are more than
// (7 + 1.22 |g|) of t, and than t itself where 2^it or its inverse has left f32's range.
constexpr float kGateError = 20 * 0x1p-24f, kFarGateError = 0.05f * 0x1p-24f;
__device__ __forceinline__ float gated32(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f)) * u;
}

template <int TYPE, int CHUNKS>
__global__ __launch_bounds__(64 * kMostWaves) void swiglu_rows_kernel(RowArgs a) {
    __shared__ double lds[kMostWaves][2];
    __shared__ float tops[2][kMostWaves];
    __shared__ unsigned long long largest[2];  // bits of a number that is not negative
    const int first = 8 * threadIdx.x, step = 8 * blockDim.x, waves = (blockDim.x + 63) >> 6;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x, turn ^= 1) {
        auto place = [&](int b) { return first + (b >> 3) * step + (b & 7); };  // in the row, of a thread's value b
        auto exact = [&](int i) {
            if (i >= a.n) return 0.0;
            return gated_value(value_at(a.x, TYPE, row * a.x_stride + i), value_at(a.y, TYPE, row * a.y_stride + i));
        };
        float t[CHUNKS][8], top = 0.0f, wide = 0.0f;
        {
            typename RowElem<TYPE>::Raw8 g[CHUNKS], u[CHUNKS];
            load_row<TYPE, CHUNKS>(row_at(a.x, TYPE, row * a.x_stride), a.n, g);
            load_row<TYPE, CHUNKS>(row_at(a.y, TYPE, row * a.y_stride), a.n, u);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = static_cast<float>(u[c][j]);
                    t[c][j] = gated32(static_cast<float>(g[c][j]), y);
                    top = __builtin_elementwise_maximum(top, fabsf(t[c][j]));  // NaN stays
                    wide = fmaxf(wide, fabsf(y));
                }
        }
        // the row's largest in f32, infinite where f32 will not do
        const float wave_top = wave_max(top == top ? top : INFINITY);
        if ((threadIdx.x & 63) == 0) tops[turn][threadIdx.x >> 6] = wave_top;
        if (threadIdx.x == 0) largest[turn] = 0;
        __syncthreads();
        float all = 0.0f;
        for (int w = 0; w < waves; ++w) all = fmaxf(all, tops[turn][w]);
        uint64_t codes[CHUNKS];
        uint32_t doubt = 0;  // a bit for each of the thread's values
        double most, unit;
        bool quick = in_range(all);
        if (quick) {
            // The value or two of the row that its largest may be, in 64 bits.  A thread with
            // a u so large that t may be off by more than kGateError of the largest takes all of
            // its values, and has all codes in doubt.
            const float at_least = all * (1.0f - 4.0f * kGateError);
            const bool far = wide > 256.0f * all;
            if (top >= at_least || far) {
                uint32_t left = 0;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) left |= fabsf(t[c][j]) >= at_least ? 1u << (8 * c + j) : 0u;
                if (far) left = ~0u;
                for (; left; left &= left - 1) {
                    const int b = __builtin_ctz(left);
                    if (b >= 8 * CHUNKS) break;
                    const double x = fabs(exact(place(b)));
                    atomicMax(&largest[turn], __builtin_bit_cast(unsigned long long, x));
                }
            }
            // meanwhile the codes by the f32 one: both are off by kGateError, the quotient by 5
            // units of 2^-24
            const float unit32 = 127.0f / all;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                uint32_t d;
                codes[c] = pack_codes<true>(t[c], unit32, fmaf(kFarGateError * wide, unit32, 1e-6f),
                                            (2.0f * kGateError + 8 * 0x1p-24f) * unit32, &d);
                doubt |= d << (8 * c);
            }
            if (far) doubt = ~0u;
            __syncthreads();
            most = __builtin_bit_cast(double, largest[turn]);
            unit = 127.0 / most;
            // (the largest in f32 may be one of such a thread's)
            quick = fabs(most - all) <= all * (1.25 * kGateError);
            if (quick && threadIdx.x == 0) a.scales[row] = static_cast<float>(most / 127.0);
        }
        if (!quick) {
            double sum = most = 0.0;
            for (int i = first; i < a.n; i += step)
                for (int j = 0; j < 8; ++j) {
                    const double x = exact(i + j);
                    most = fmax(most, fabs(x));
                    sum = fma(x, 0.0, sum);  // NaN where x is not finite
                }
            group_sum_max(&sum, &most, lds);
            __syncthreads();  // lds
            const bool bad = !(fabs(sum) <= 1.7976931348623157e308), zero = bad || most == 0.0;
            unit = zero ? 0.0 : 127.0 / most;
            if (threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(most / 127.0);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) codes[c] = 0;
            doubt = zero ? 0 : ~0u;
        }
        int8_t *q = a.q + row * a.q_stride;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            row_store_codes(q, first + c * step, a.n, codes[c]);
        // codes in doubt once more
        for (; doubt; doubt &= doubt - 1) {
            const int b = __builtin_ctz(doubt), i = place(b);
            if (b < 8 * CHUNKS && i < a.n) q[i] = static_cast<int8_t>(code_of(exact(i), most, unit));
        }
    }
}

// ---- launches ------------------------------------------------------------------

// Threads, and runs of 8 values of each: as many threads as there are runs for few
// rows, so that a row's latency is short (one row of 8192 4.2 us, with 4 runs a thread
// 4.9); for many rows up to 4 runs each, so that fewer threads meet at a row's barriers,
// while 256 threads are left, or 128 where a value is much work (300 rows of 8192, one, two
// and four runs a thread 8.9, 7.9, 9.1; 8192 rows of 8192 116, 94, 91; without a residual
// 94, 56, 45; rows of 2048 26, 27, 31; 4096 gated rows of 14336 76, 76, 63; 8192 of 2048 25,
// 21, 21).
struct RowShape {
    int threads, chunks;
};
RowShape row_shape(const mi355x_ctx *ctx, const RowArgs &a, int fewest) {
    const int runs = (a.n + 7) / 8, most = 64 * kMostWaves;
    const int least = (runs + most - 1) / most;
    const int wanted = a.n_rows >= 4 * ctx->num_cus ? 4 : a.n_rows >= ctx->num_cus ? 2 : 1;
    int chunks = std::max(least, std::min(wanted, runs / fewest));
    chunks = chunks <= 1 ? 1 : chunks <= 2 ? 2 : 4;
    return {std::min(most, ((runs + chunks - 1) / chunks + 63) / 64 * 64), chunks};
}

template <class F>
int by_chunks(int chunks, F f) {
    if (chunks == 1) return f(std::integral_constant<int, 1>{});
    if (chunks == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 4>{});
}

unsigned row_groups(const RowArgs &a) { return static_cast<unsigned>(std::min<int64_t>(a.n_rows, 1 << 20)); }

template <bool GATED>
int launch_long(mi355x_ctx *ctx, const RowArgs &a) {
    row_q8_kernel<GATED><<<row_groups(a), 64 * kMostWaves, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

template <int XT, int RT>
int launch_norm(mi355x_ctx *ctx, const RowArgs &a) {
    const RowShape s = row_shape(ctx, a, 256);
    unsigned groups = row_groups(a);
    if (s.chunks > 1) {  // workgroups keep the norm's weights over several rows (8192 rows of 8192: 91 us, 95 without)
        const int64_t per = (a.n_rows + 8 * ctx->num_cus - 1) / (8 * ctx->num_cus);
        groups = static_cast<unsigned>(std::min<int64_t>(groups, (a.n_rows + per - 1) / per));
    }
    return by_chunks(s.chunks, [&](auto c) {
        norm_rows_kernel<XT, RT, decltype(c)::value><<<groups, s.threads, 0, ctx->stream>>>(a);
        MI355X_HIP(hipGetLastError());
        return MI355X_OK;
    });
}

template <int XT>
int launch_norm_of(mi355x_ctx *ctx, const RowArgs &a) {
    if (!a.y) return launch_norm<XT, -1>(ctx, a);
    if (a.residual_type == MI355X_TYPE_F32) return launch_norm<XT, MI355X_TYPE_F32>(ctx, a);
    if (a.residual_type == MI355X_TYPE_F16) return launch_norm<XT, MI355X_TYPE_F16>(ctx, a);
    return launch_norm<XT, MI355X_TYPE_BF16>(ctx, a);
}

template <int TYPE>
int launch_swiglu(mi355x_ctx *ctx, const RowArgs &a) {
    const RowShape s = row_shape(ctx, a, 128);
    return by_chunks(s.chunks, [&](auto c) {
        swiglu_rows_kernel<TYPE, decltype(c)::value><<<row_groups(a), s.threads, 0, ctx->stream>>>(a);
        MI355X_HIP(hipGetLastError());
        return MI355X_OK;
    });
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
    if (a.n > kMostHeld) return launch_long<false>(ctx, a);
    if (a.type == MI355X_TYPE_F32) return launch_norm_of<MI355X_TYPE_F32>(ctx, a);
    if (a.type == MI355X_TYPE_F16) return launch_norm_of<MI355X_TYPE_F16>(ctx, a);
    return launch_norm_of<MI355X_TYPE_BF16>(ctx, a);
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
    if (a.n > kMostHeld) return launch_long<true>(ctx, a);
    if (a.type == MI355X_TYPE_F32) return launch_swiglu<MI355X_TYPE_F32>(ctx, a);
    if (a.type == MI355X_TYPE_F16) return launch_swiglu<MI355X_TYPE_F16>(ctx, a);
    return launch_swiglu<MI355X_TYPE_BF16>(ctx, a);
}

}  // namespace mi355x
