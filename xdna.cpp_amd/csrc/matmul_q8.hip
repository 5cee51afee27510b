// Products of 8-bit integers with a scale for each row and each channel, on the
// integer matrix cores: sums of products of codes are exact in 32 bits (128 * 128
// * 131056 < 2^31), so the order of the sum and the split of the work do not show.
//
// The weight is the products' left operand: a lane then holds consecutive channels
// of one row of the output.
#include "far_parts.h"
#include "internal.h"

#include <algorithm>

namespace mi355x {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct MatmulArgs {
    int64_t x_stride, w_stride, out_stride;
    const int8_t *x, *w;
    const float *x_scales, *w_scales, *bias;
    void *out;
    int *counters;  // 0 before and after a call
    float *ws;
    int m, n, k, out_type;
    int wide;            // stores of four channels at once keep to their alignment
    int m_tiles, n_tiles, splits, split_steps;
};

constexpr int kStepBytes = 64;  // of k that one matrix product takes

__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// One value of the product, in the stated order of roundings.
__device__ __forceinline__ float scaled(int sum, float ws, float xs, bool has_bias, float bias) {
#pragma clang fp contract(off)
    float v = static_cast<float>(sum) * ws;
    v = v * xs;
    if (has_bias) v = v + bias;
    return v;
}

template <class T>
__device__ __forceinline__ void store4(void *out, int64_t at, int left, bool wide, const float *v) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T *p = static_cast<T *>(out) + at;
    if (wide && left >= 4) {
        *reinterpret_cast<T4 *>(p) = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = static_cast<T>(v[i]);
    }
}

// Channels n .. n + 3 of row m from their sums.
__device__ __forceinline__ void write4(const MatmulArgs &a, int m, int n, i32x4 sum) {
    if (m >= a.m || n >= a.n) return;
    const float xs = a.x_scales[m];
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = min(n + i, a.n - 1);
        v[i] = scaled(sum[i], a.w_scales[c], xs, a.bias != nullptr, a.bias ? a.bias[c] : 0.0f);
    }
    const int64_t at = m * a.out_stride + n;
    if (a.out_type == MI355X_TYPE_F32) store4<float>(a.out, at, a.n - n, a.wide, v);
    else if (a.out_type == MI355X_TYPE_F16) store4<_Float16>(a.out, at, a.n - n, a.wide, v);
    else store4<__bf16>(a.out, at, a.n - n, a.wide, v);
}

// ---- few rows ------------------------------------------------------------------

// A workgroup computes 16 * R channels of up to 16 * TM rows; its wavefronts share
// out k and add their sums in LDS.
constexpr int kFewWaves = 8;

template <int TM, int R>
__global__ __launch_bounds__(64 * kFewWaves) void matmul_few_kernel(MatmulArgs a) {
    constexpr int U = TM >= 3 ? 2 : 4;  // steps whose operands are loaded together
    __shared__ i32x4 part[kFewWaves][R * TM][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16 * R, m0 = blockIdx.y * 16 * TM;
    const int steps = (a.k + kStepBytes - 1) / kStepBytes;
    const int s0 = steps * wave / kFewWaves, s1 = steps * (wave + 1) / kFewWaves;
    const int8_t *w[R], *x[TM];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = a.w + static_cast<int64_t>(min(n0 + 16 * r + col, a.n - 1)) * a.w_stride;
#pragma unroll
    for (int t = 0; t < TM; ++t) x[t] = a.x + static_cast<int64_t>(min(m0 + 16 * t + col, a.m - 1)) * a.x_stride;
    i32x4 c[R][TM];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TM; ++t) c[r][t] = i32x4{0, 0, 0, 0};
    i32x4 wf[2][U][R], xf[2][U][TM];
    auto load = [&](int b, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = kStepBytes * (s + u) + 16 * quad;
            const bool in = s + u < s1 && k < a.k;
            const int at = in ? k : 0;
#pragma unroll
            for (int r = 0; r < R; ++r) wf[b][u][r] = *reinterpret_cast<const i32x4 *>(w[r] + at);
#pragma unroll
            for (int t = 0; t < TM; ++t) xf[b][u][t] = *reinterpret_cast<const i32x4 *>(x[t] + at);
        }
    };
    auto multiply = [&](int b, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = s + u < s1 && kStepBytes * (s + u) + 16 * quad < a.k;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                i32x4 v = wf[b][u][r];
                if (!in) v = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < TM; ++t) c[r][t] = mfma(v, xf[b][u][t], c[r][t]);
            }
        }
    };
    if (s0 < s1) {
        load(0, s0);
        for (int s = s0; s < s1; s += 2 * U) {
            if (s + U < s1) load(1, s + U);
            multiply(0, s);
            if (s + U < s1) {
                if (s + 2 * U < s1) load(0, s + 2 * U);
                multiply(1, s + U);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TM; ++t) part[wave][r * TM + t][lane] = c[r][t];
    __syncthreads();
    for (int b = wave; b < R * TM; b += kFewWaves) {
        i32x4 sum = part[0][b][lane];
#pragma unroll
        for (int v = 1; v < kFewWaves; ++v) sum += part[v][b][lane];
        write4(a, m0 + 16 * (b % TM) + col, n0 + 16 * (b / TM) + 4 * quad, sum);
    }
}

// ---- many rows -------------------------------------------------------------------

// A workgroup computes BM rows by BN channels from tiles in LDS.  Such tiles travel
// there directly (global_load_lds), kStages - 1 steps ahead; a load fills 16 rows of
// 64 bytes in lane order, four lanes a row, whose 16-byte chunks are permuted by the
// row's number so that the operands' reads (16 rows, one chunk) do not meet in a bank.
constexpr int kStages = 4;

template <int BM, int BN, int WM, int WN>
struct TileShape {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int kBlocks = (BM + BN) / 16;       // of a stage, 1 KB each
    static constexpr int kLoads = kBlocks / kWaves;      // of a wavefront and stage
    static constexpr int kStageBytes = 1024 * kBlocks;
    static constexpr int kLds = kStages * kStageBytes;
    static constexpr int kPartInts = BM * BN;
    static_assert(kBlocks % kWaves == 0, "every wavefront loads as many blocks");
};

// The tile that workgroup `id` of `total` computes: each die (workgroups go round
// the 8 dies) takes a run of them, rows first within bands of 8 row tiles, so that
// what it reads stays in its L2.
__device__ __forceinline__ void tile_of(const MatmulArgs &a, int id, int total, int *mt, int *nt, int *split) {
    const int die = id & 7, each = total >> 3, over = total & 7;
    int t = die * each + min(die, over) + (id >> 3);
    const int tiles = a.m_tiles * a.n_tiles;
    *split = t / tiles;
    t -= *split * tiles;
    const int band = t / (8 * a.n_tiles);
    const int rows = min(8, a.m_tiles - 8 * band);
    t -= 8 * band * a.n_tiles;
    *nt = t / rows;
    *mt = 8 * band + t - *nt * rows;
}

template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void matmul_tile_kernel(MatmulArgs a) {
    typedef TileShape<BM, BN, WM, WN> S;
    constexpr int TM = S::TM, TN = S::TN;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    int mt, nt, split;
    tile_of(a, blockIdx.x, gridDim.x, &mt, &nt, &split);
    const int m0 = mt * BM, n0 = nt * BN;
    const int steps = (a.k + kStepBytes - 1) / kStepBytes;
    const int s0 = split * a.split_steps, s1 = min(steps, s0 + a.split_steps);

    // blocks of a stage: BN / 16 of w, then BM / 16 of x
    const int8_t *src[S::kLoads];
    const int chunk = 16 * ((lane & 3) ^ (lane >> 4)), r = lane >> 2;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
        const int b = wave * S::kLoads + i;
        if (b < BN / 16) {
            // a wavefront's channels are dealt out so that a lane's are consecutive
            const int wn = b / TN, tn = b % TN;
            const int n = n0 + wn * 16 * TN + (r >> 2) * 4 * TN + 4 * tn + (r & 3);
            src[i] = a.w + static_cast<int64_t>(min(n, a.n - 1)) * a.w_stride;
        } else {
            const int m = m0 + 16 * (b - BN / 16) + r;
            src[i] = a.x + static_cast<int64_t>(min(m, a.m - 1)) * a.x_stride;
        }
    }
    auto load = [&](int s) {
        const int k = kStepBytes * s + chunk;
        const int at = k < a.k ? k : 0;
        uint8_t *dst = lds + (s - s0) % kStages * S::kStageBytes + 1024 * wave * S::kLoads;
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i)
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(reinterpret_cast<uintptr_t>(src[i] + at)),
                (__attribute__((address_space(3))) uint32_t *)(dst + 1024 * i), 16, 0, 0);
    };
    i32x4 c[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) c[i][j] = i32x4{0, 0, 0, 0};
    const int wm = wave % WM, wn = wave / WM;
    const int slot = 16 * (4 * col + (quad ^ (col >> 2)));
    const int w_at = 1024 * wn * TN + slot, x_at = 1024 * (BN / 16 + wm * TM) + slot;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (s0 + i < s1) load(s0 + i);
    for (int s = s0; s < s1; ++s) {
        // this wavefront's loads of stage s are done where only the later ones are left
        if (s + kStages - 2 < s1) __builtin_amdgcn_s_waitcnt(0x0F70 | ((kStages - 2) * S::kLoads));
        else __builtin_amdgcn_s_waitcnt(0x0F70);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + kStages - 1 < s1) load(s + kStages - 1);
        const uint8_t *stage = lds + (s - s0) % kStages * S::kStageBytes;
        i32x4 wf[TN], xf[TM];
#pragma unroll
        for (int i = 0; i < TN; ++i) wf[i] = *reinterpret_cast<const i32x4 *>(stage + w_at + 1024 * i);
#pragma unroll
        for (int j = 0; j < TM; ++j) xf[j] = *reinterpret_cast<const i32x4 *>(stage + x_at + 1024 * j);
        if (kStepBytes * s + 16 * quad >= a.k)
#pragma unroll
            for (int i = 0; i < TN; ++i) wf[i] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i) c[i][j] = mfma(wf[i], xf[j], c[i][j]);
    }
    if (a.splits > 1) {
        const FarParts far(a.ws);
        const int tile = mt * a.n_tiles + nt, tiles = a.m_tiles * a.n_tiles;
        const int mine = 4 * (wave * TM * TN * 64 + lane);
        const int at = (split * tiles + tile) * S::kPartInts + mine;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) far.store4(at + 256 * (i * TM + j), __builtin_bit_cast(f32x4, c[i][j]));
        if (!last_of(a.counters + tile, a.splits, reinterpret_cast<int *>(lds))) return;
        for (int p = 0; p < a.splits; ++p) {
            if (p == split) continue;
            const int from = (p * tiles + tile) * S::kPartInts + mine;
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) c[i][j] += __builtin_bit_cast(i32x4, far.load4(from + 256 * (i * TM + j)));
        }
    }
    const int n = n0 + wn * 16 * TN + quad * 4 * TN, m = m0 + wm * 16 * TM + col;
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i) write4(a, m + 16 * j, n + 4 * i, c[i][j]);
}

// ---- the choice ---------------------------------------------------------------

constexpr size_t kCounters = 4096;
constexpr size_t kPartBytes = size_t(64) << 20;

template <int TM, int R>
int launch_few(mi355x_ctx *ctx, const MatmulArgs &a) {
    matmul_few_kernel<TM, R><<<(a.n + 16 * R - 1) / (16 * R), 64 * kFewWaves, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

template <int BM, int BN, int WM, int WN>
int launch_tiles(mi355x_ctx *ctx, MatmulArgs a) {
    typedef TileShape<BM, BN, WM, WN> S;
    static bool sized = false;  // the same for every device
    if (!sized) {
        MI355X_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(matmul_tile_kernel<BM, BN, WM, WN>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds));
        sized = true;
    }
    a.m_tiles = (a.m + BM - 1) / BM;
    a.n_tiles = (a.n + BN - 1) / BN;
    const int64_t tiles = static_cast<int64_t>(a.m_tiles) * a.n_tiles;
    if (tiles >= (1 << 22))
        return set_error(MI355X_EUNSUPPORTED,
                         "mi355x_matmul_q8: " + std::to_string(tiles) + " tiles of the output, 2^22 or more");
    const int steps = (a.k + kStepBytes - 1) / kStepBytes;
    int64_t splits = 1;
    if (tiles <= ctx->num_cus / 2)
        splits = std::min<int64_t>({ctx->num_cus / tiles, steps / 16, int64_t(kPartBytes / (4 * S::kPartInts) / tiles)});
    splits = std::max<int64_t>(splits, 1);
    a.split_steps = static_cast<int>((steps + splits - 1) / splits);
    a.splits = (steps + a.split_steps - 1) / a.split_steps;
    matmul_tile_kernel<BM, BN, WM, WN>
        <<<static_cast<unsigned>(tiles * a.splits), S::kThreads, S::kLds, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace

size_t matmul_q8_workspace_bytes(const mi355x_ctx *) { return kCounters + kPartBytes; }

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
    a.counters = static_cast<int *>(u.workspace);
    a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(u.workspace) + kCounters);
    a.m = static_cast<int>(u.n_rows);
    a.n = static_cast<int>(u.n_out);
    a.k = static_cast<int>(u.k);
    a.out_type = u.out_type;
    const int64_t four = u.out_type == MI355X_TYPE_F32 ? 16 : 8;
    a.wide = reinterpret_cast<uintptr_t>(u.out) % four == 0 && u.out_stride % 4 == 0;
    if (a.m <= 16) return a.n > 8192 ? launch_few<1, 2>(ctx, a) : launch_few<1, 1>(ctx, a);
    if (a.m <= 32) return launch_few<2, 2>(ctx, a);
    if (a.m <= 48) return launch_few<3, 2>(ctx, a);
    if (a.m <= 64) return launch_few<4, 2>(ctx, a);
    const int64_t large = static_cast<int64_t>((a.m + 255) / 256) * ((a.n + 255) / 256);
    if (large >= ctx->num_cus) return launch_tiles<256, 256, 2, 4>(ctx, a);
    return launch_tiles<128, 128, 2, 2>(ctx, a);
}

}  // namespace mi355x
