// Products of 8-bit integers with a scale for each row and each channel, on the
// integer matrix cores: sums of products of codes are exact in 32 bits (128 * 128
// * 131056 < 2^31), so the order of the sum and the split of the work do not show.
//
// The weight is the products' left operand: a lane then holds four consecutive
// channels of one row of the output.
//
// All operands travel to LDS directly (global_load_lds, whole 128-byte lines) in
// pieces of 8 rows, eight lanes a row; such loads fill LDS in lane order, so the
// 16-byte chunks of a row are permuted by the row's number, that the operands' reads
// (16 rows, one chunk) do not meet in a bank.
#include "far_parts.h"
#include "internal.h"
#include "matmul_q8_forms.h"
#include "paged_index.h"

#include <algorithm>

namespace mi355x {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kCounterStep = 32;  // ints from one tile's counter to the next: a cache line

struct MatmulArgs {
    int64_t x_stride, w_stride, out_stride;
    const int8_t *x, *w;
    const float *x_scales, *w_scales, *bias;
    void *out;
    int *counters;  // 0 before and after a call
    float *ws;
    int m, n, k, out_type;
    int m_tiles, n_tiles, splits, split_stages;
    FastDiv tiles, band, last_rows;  // m_tiles * n_tiles, 8 * n_tiles, m_tiles % 8 (or 8)
};

constexpr int kStage = kMatmulStage;  // bytes of k in a stage: two matrix products deep

__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// At most N of this wavefront's loads (and stores) are under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
}
// The same, and all of its LDS reads are done.
template <int N>
__device__ __forceinline__ void wait_loads_and_reads() {
    static_assert(N >= 0 && N < 64, "");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
}
__device__ __forceinline__ void wait_reads() { __builtin_amdgcn_s_waitcnt(0xC07F); }

__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Row `row` (0 .. 7 of the piece's half, 8 more for the second) and chunk of a piece
// that a lane fills, and where an operand's lane finds its chunk again.
__device__ __forceinline__ int piece_row(int half, int lane) { return 8 * half + (lane >> 3); }
__device__ __forceinline__ int piece_chunk(int half, int lane) {
    return 16 * ((lane & 7) ^ (piece_row(half, lane) >> 1));
}
__device__ __forceinline__ int operand_at(int half, int col, int quad) {
    return 128 * col + 16 * ((4 * half + quad) ^ (col >> 1));
}

// One value of the product, in the stated order of roundings.
__device__ __forceinline__ float scaled(int sum, float ws, float xs, bool has_bias, float bias) {
#pragma clang fp contract(off)
    float v = static_cast<float>(sum) * ws;
    v = v * xs;
    if (has_bias) v = v + bias;
    return v;
}

template <class T, int N>
__device__ __forceinline__ void store_some(void *out, int64_t at, int left, const float *v) {
    typedef T TN __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    T *p = static_cast<T *>(out) + at;
    if (left >= N) {
        TN t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = static_cast<T>(v[i]);
        *reinterpret_cast<TN *>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = static_cast<T>(v[i]);
    }
}

// Channels n .. n + N - 1 of row m.
template <int N>
__device__ __forceinline__ void store_row(const MatmulArgs &a, int m, int n, const float *v) {
    const int64_t at = m * a.out_stride + n;
    if (a.out_type == MI355X_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) store_some<float, 4>(a.out, at + i, a.n - n - i, v + i);
    } else if (a.out_type == MI355X_TYPE_F16) {
        store_some<_Float16, N>(a.out, at, a.n - n, v);
    } else {
        store_some<__bf16, N>(a.out, at, a.n - n, v);
    }
}

// Number n of a vector of `size` (the last one where it is behind it), from a uniform base.
__device__ __forceinline__ float one_of(const float *p, int n, int size) {
    const uint32_t at = 4u * static_cast<uint32_t>(min(n, size - 1));
    return *reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(p) + at);
}
// Four of them from n on.
__device__ __forceinline__ f32x4 four_of(const float *p, int n, int size) {
    return f32x4{one_of(p, n, size), one_of(p, n + 1, size), one_of(p, n + 2, size), one_of(p, n + 3, size)};
}
// A bias's numbers are asked for without a branch, of the scales where there is none.
__device__ __forceinline__ const float *bias_or_scales(const MatmulArgs &a) { return a.bias ? a.bias : a.w_scales; }

// ---- few rows ------------------------------------------------------------------

// A workgroup computes 16 * R channels of up to 16 * TM rows.  Its WAVES wavefronts
// share out k, each with a ring of ST stages of its own, and add their sums in LDS, so
// that no wavefront waits for another while weights stream.  Bound by memory, with weights
// taken in turn from 1.1 GB of them: one row of 22016 channels, k 2048, 45 MB, 10.2 us (4.4
// TB/s); of 151936 52 us (6.0); 32 rows of 28672, k 4096 26.7 us (4.5).  One weight over and
// over, which the last-level cache holds where it is below 256 MB: 7.6, 48, 19.1.  Not so
// for few channels: one row of 2048, k 11008 7.4 us (3.0 TB/s; 5.5), as 128 workgroups leave half
// of the CUs without one.
template <int TM, int R, int WAVES, int ST>
struct FewShape {
    static constexpr int kUnit = 2048 * (TM + R);
    static constexpr int kRing = WAVES * ST * kUnit, kSums = WAVES * R * TM * 1024;
    static constexpr int kLds = kRing > kSums ? kRing : kSums;
};

template <int TM, int R, int WAVES, int ST>
__global__ __launch_bounds__(64 * WAVES) void matmul_few_kernel(MatmulArgs a) {
    typedef FewShape<TM, R, WAVES, ST> S;
    constexpr int kBlocks = R + TM, kLoads = 2 * kBlocks;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16 * R, m0 = blockIdx.y * 16 * TM;
    const int stages = (a.k + kStage - 1) / kStage;
    const int s0 = stages * wave / WAVES, s1 = stages * (wave + 1) / WAVES;
    const int8_t *src[kBlocks][2];
    int chunk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        chunk[i] = piece_chunk(i, lane);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const int row = 16 * (b < R ? b : b - R) + piece_row(i, lane);
            src[b][i] = (b < R ? a.w + min(n0 + row, a.n - 1) * a.w_stride : a.x + min(m0 + row, a.m - 1) * a.x_stride) +
                        chunk[i];
        }
    }
    // the scales of the wavefront's first block of outputs are asked for before the codes
    const int m_first = m0 + 16 * (wave % TM) + col, n_first = n0 + 16 * (wave / TM) + 4 * quad;
    float xs = one_of(a.x_scales, m_first, a.m);
    f32x4 ws = four_of(a.w_scales, n_first, a.n), bias = four_of(bias_or_scales(a), n_first, a.n);
    uint8_t *mine = lds + wave * ST * S::kUnit;
    auto load = [&](int s, int slot) {
        const int k = kStage * s;
        int at[2] = {k, k};
        if (k + kStage > a.k)  // instead of chunks behind the rows' ends the stage's first
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (k + chunk[i] >= a.k) at[i] = k - chunk[i];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                __builtin_amdgcn_global_load_lds(
                    reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(
                        reinterpret_cast<uintptr_t>(src[b][i] + at[i])),
                    (__attribute__((address_space(3))) uint32_t *)(mine + slot * S::kUnit + 2048 * b + 1024 * i), 16, 0, 0);
    };
    i32x4 c[R][TM];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TM; ++t) c[r][t] = i32x4{0, 0, 0, 0};
    auto multiply = [&](int s, int slot) {
        i32x4 f[2][kBlocks];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                f[h][b] = *reinterpret_cast<const i32x4 *>(mine + slot * S::kUnit + 2048 * b + operand_at(h, col, quad));
        if (kStage * (s + 1) > a.k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (kStage * s + 64 * h + 16 * quad >= a.k)
#pragma unroll
                    for (int r = 0; r < R; ++r) f[h][r] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < TM; ++t) c[r][t] = mfma(f[h][r], f[h][R + t], c[r][t]);
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i)
        if (s0 + i < s1) load(s0 + i, i);
    int slot = 0;
    for (int s = s0; s < s1; ++s) {
        // the slot that is filled was read in the last step, whose products have its values
        if (s + ST - 1 < s1) {
            load(s + ST - 1, slot == 0 ? ST - 1 : slot - 1);
            wait_loads<(ST - 1) * kLoads>();
        } else {
            wait_loads<0>();
        }
        asm volatile("" ::: "memory");
        multiply(s, slot);
        wait_reads();
        asm volatile("" ::: "memory");
        slot = slot + 1 == ST ? 0 : slot + 1;
    }
    __syncthreads();
    i32x4 *sums = reinterpret_cast<i32x4 *>(lds);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TM; ++t) sums[(wave * R * TM + r * TM + t) * 64 + lane] = c[r][t];
    __syncthreads();
    for (int b = wave; b < R * TM; b += WAVES) {
        i32x4 sum = sums[b * 64 + lane];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += sums[(v * R * TM + b) * 64 + lane];
        const int m = m0 + 16 * (b % TM) + col, n = n0 + 16 * (b / TM) + 4 * quad;
        if (b != wave) {
            xs = one_of(a.x_scales, m, a.m);
            ws = four_of(a.w_scales, n, a.n);
            bias = four_of(bias_or_scales(a), n, a.n);
        }
        if (m < a.m && n < a.n) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = scaled(sum[i], ws[i], xs, a.bias != nullptr, bias[i]);
            store_row<4>(a, m, n, v);
        }
    }
}

// ---- tiles -------------------------------------------------------------------

// The tile that workgroup `id` of `total` computes: each die (workgroups go round
// the 8 dies) takes a run of them, rows first within bands of 8 row tiles, so that
// what it reads stays in its L2.
__device__ __forceinline__ void tile_of(const MatmulArgs &a, int id, int total, int *mt, int *nt, int *split) {
    const int die = id & 7, each = total >> 3, over = total & 7;
    int t = die * each + min(die, over) + (id >> 3);
    *split = divided(t, a.tiles);
    t -= *split * static_cast<int>(a.tiles.d);
    const int band = divided(t, a.band);
    t -= band * static_cast<int>(a.band.d);
    if (8 * band + 8 <= a.m_tiles) {
        *nt = t >> 3;
        *mt = 8 * band + (t & 7);
    } else {
        *nt = divided(t, a.last_rows);
        *mt = 8 * band + t - *nt * static_cast<int>(a.last_rows.d);
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const int8_t *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p), 0, 0xFFFFFFFFu, kBufferWord3);
}
__device__ __forceinline__ void load_piece(__amdgpu_buffer_rsrc_t rows, uint8_t *dst, uint32_t at, uint32_t k) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (__attribute__((address_space(3))) void *)dst, 16, at, k, 0, 0);
}

// Channel of a wavefront that row `row` of its block `tn` of 16 stands for.  For a
// 16-bit output two blocks share 32 channels so that a lane has 8 consecutive ones.
__device__ __forceinline__ int channel_of(int row, int tn, bool pairs) {
    return pairs ? 32 * (tn >> 1) + 8 * (row >> 2) + 4 * (tn & 1) + (row & 3) : 16 * tn + row;
}

// The scales of a wavefront's outputs: rows m + 16 j, channels from n on.
template <int TM, int TN>
struct TileScales {
    f32x4 w[TN], bias[TN];
    float x[TM];
    __device__ __forceinline__ TileScales(const MatmulArgs &a, int m, int n, int quad) {
        const bool pairs = a.out_type != MI355X_TYPE_F32;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int ch = n + channel_of(4 * quad, i, pairs);
            w[i] = four_of(a.w_scales, ch, a.n);
            bias[i] = four_of(bias_or_scales(a), ch, a.n);
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) x[j] = one_of(a.x_scales, m + 16 * j, a.m);
    }
};

template <int TM, int TN>
__device__ __forceinline__ void write_tile(const MatmulArgs &a, int m, int n, const i32x4 (&c)[TN][TM], int quad,
                                           const TileScales<TM, TN> &scales) {
    const bool pairs = a.out_type != MI355X_TYPE_F32, has_bias = a.bias != nullptr;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int row = m + 16 * j;
        if (row >= a.m) continue;
#pragma unroll
        for (int i = 0; i < TN; i += 2) {
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                v[q] = scaled(c[i + q / 4][j][q % 4], scales.w[i + q / 4][q % 4], scales.x[j], has_bias,
                              scales.bias[i + q / 4][q % 4]);
            if (pairs) {
                const int ch = n + channel_of(4 * quad, i, true);
                if (ch < a.n) store_row<8>(a, row, ch, v);
            } else {
                const int ch = n + channel_of(4 * quad, i, false);
                if (ch < a.n) store_row<4>(a, row, ch, v);
                if (ch + 16 < a.n) store_row<4>(a, row, ch + 16, v + 4);
            }
        }
    }
}

// A workgroup of WM x WN wavefronts computes BM rows by BN channels from a ring of ST
// stages.  One barrier a stage; operands are read half a stage ahead of their
// products.  Where there are few tiles k is split, and the last workgroup of a tile
// adds the others' sums to its own.  Most of the time goes to operands on their way from
// L2 to LDS: each stage brings BM + BN rows for BM * BN products, at about 48 GB/s a CU
// (12.3 TB/s in all) however many stages are under way.  That is what this loop gets and no
// limit of L2: the same loads without products run at 12 to 18 TB/s.  512 x 4096, k 14336,
// 128 x 128 in 2 parts: 41 us with one weight over and over, 45 with weights in turn from
// memory (1.4 Pop/s), 531 MB from L2; parts and their join are 5 us.  Rows 128, 256 and 384 bytes
// further apart, which spreads a stage's lines over other channels of L2: 41, 44.
template <int BM, int BN, int WM, int WN, int ST>
struct TileShape {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int kBlocks = (BM + BN) / 16;
    static constexpr int kLoads = 2 * kBlocks / kWaves;  // pieces of a wavefront and stage
    static constexpr int kStageBytes = 2048 * kBlocks;
    static constexpr int kLds = ST * kStageBytes;
    static_assert(2 * kBlocks % kWaves == 0 && TN % 2 == 0, "");
};

template <int BM, int BN, int WM, int WN, int ST>
__global__ __launch_bounds__(64 * WM * WN) void matmul_tile_kernel(MatmulArgs a) {
    typedef TileShape<BM, BN, WM, WN, ST> S;
    constexpr int TM = S::TM, TN = S::TN;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    int mt, nt, split;
    tile_of(a, blockIdx.x, gridDim.x, &mt, &nt, &split);
    const int m0 = mt * BM, n0 = nt * BN;
    const int s0 = split * a.split_stages, s1 = min((a.k + kStage - 1) / kStage, s0 + a.split_stages);
    const bool pairs = a.out_type != MI355X_TYPE_F32;
    const __amdgpu_buffer_rsrc_t w_rows = rows_at(a.w + n0 * a.w_stride), x_rows = rows_at(a.x + m0 * a.x_stride);
    // blocks of a stage: BN / 16 of w, then BM / 16 of x
    uint32_t at[S::kLoads];
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
        const int p = wave * S::kLoads + i, b = p >> 1, row = piece_row(p & 1, lane);
        const uint32_t r = b < BN / 16 ? min(16 * TN * (b / TN) + channel_of(row, b % TN, pairs), a.n - 1 - n0)
                                       : min(16 * (b - BN / 16) + row, a.m - 1 - m0);
        at[i] = r * static_cast<uint32_t>(b < BN / 16 ? a.w_stride : a.x_stride) + piece_chunk(p & 1, lane);
    }
    auto load = [&](int s, int slot) {
        const int k = kStage * s;
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const int p = wave * S::kLoads + i;
            uint32_t v = at[i];
            if (k + kStage > a.k && k + piece_chunk(p & 1, lane) >= a.k) v -= piece_chunk(p & 1, lane);
            if (p < BN / 8) load_piece(w_rows, lds + slot * S::kStageBytes + 1024 * p, v, k);
            else load_piece(x_rows, lds + slot * S::kStageBytes + 1024 * p, v, k);
        }
    };
    const int wm = wave % WM, wn = wave / WM;
    const int w_at = 2048 * wn * TN, x_at = 2048 * (BN / 16 + wm * TM);
    i32x4 c[TN][TM], wf[2][TN], xf[2][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) c[i][j] = i32x4{0, 0, 0, 0};
    auto read = [&](int h, int slot) {
        const uint8_t *p = lds + slot * S::kStageBytes + operand_at(h, col, quad);
#pragma unroll
        for (int i = 0; i < TN; ++i) wf[h][i] = *reinterpret_cast<const i32x4 *>(p + w_at + 2048 * i);
#pragma unroll
        for (int j = 0; j < TM; ++j) xf[h][j] = *reinterpret_cast<const i32x4 *>(p + x_at + 2048 * j);
    };
    auto multiply = [&](int h) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int i = 0; i < TN; ++i) c[i][j] = mfma(wf[h][i], xf[h][j], c[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };
    const TileScales<TM, TN> scales(a, m0 + wm * 16 * TM + col, n0 + wn * 16 * TN, quad);
#pragma unroll
    for (int i = 0; i < ST; ++i)
        if (s0 + i < s1) load(s0 + i, i);
    // the first stage is there
    if (s0 + ST <= s1) wait_loads<(ST - 1) * S::kLoads>();
    else wait_loads<0>();
    barrier();
    // stages that k fills, then what is left of it
    const int s_whole = min(s1, a.k / kStage);
    if (s0 < s_whole) read(0, 0);
    int slot = 0;
    for (int s = s0; s < s_whole; ++s) {
        const int next = slot + 1 == ST ? 0 : slot + 1;
        read(1, slot);
        multiply(0);
        // stage s + 1 is there (up to s + ST - 1 have been asked for), and stage s has been read
        if (s + ST - 1 < s1) wait_loads_and_reads<(ST - 2) * S::kLoads>();
        else wait_loads_and_reads<0>();
        barrier();
        if (s + ST < s1) load(s + ST, slot);
        if (s + 1 < s_whole) read(0, next);
        multiply(1);
        slot = next;
    }
    if (s_whole < s1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            read(h, slot);
            if (kStage * s_whole + 64 * h + 16 * quad >= a.k)
#pragma unroll
                for (int i = 0; i < TN; ++i) wf[h][i] = i32x4{0, 0, 0, 0};
            multiply(h);
        }
    }
    if (a.splits > 1) {
        const FarParts far(a.ws);
        const int tile = mt * a.n_tiles + nt, tiles = a.m_tiles * a.n_tiles;
        const int mine = 4 * (wave * TM * TN * 64 + lane);
        const int to = (split * tiles + tile) * BM * BN + mine;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) far.store4(to + 256 * (i * TM + j), __builtin_bit_cast(f32x4, c[i][j]));
        if (!last_of(a.counters + kCounterStep * tile, a.splits, reinterpret_cast<int *>(lds))) return;
        for (int p = 0; p < a.splits; ++p) {
            if (p == split) continue;
            const int from = (p * tiles + tile) * BM * BN + mine;
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) c[i][j] += __builtin_bit_cast(i32x4, far.load4(from + 256 * (i * TM + j)));
        }
    }
    write_tile<TM, TN>(a, m0 + wm * 16 * TM + col, n0 + wn * 16 * TN, c, quad, scales);
}

// ---- large tiles -----------------------------------------------------------------

// 256 rows by 256 channels, eight wavefronts of 128 by 64 in two groups of four, one
// of each group on a SIMD.  A group's memory part (reads of a quarter of the next
// products' operands, loads of a quarter of the stage after next) runs while the other
// group multiplies; barriers swap them.  A stage is four such turns: with X0, X1 and W0,
// W1 the halves of a wavefront's rows and channels, X0 W0, X0 W1, X1 W1, X1 W0.  Of the
// two stages in LDS a quarter is free as soon as both groups have read it, so that loads
// are under way for 7 turns.  The workgroup goes through several tiles; the first
// stages of the next are loaded while a tile's outputs are written.  8192 x 8192, k 8192:
// 426 us, 2.58 Pop/s, with weights in turn 441, 2.49 (torch's library product 440 to 465;
// products alone, without loads, 262), the matrix cores busy 58% of the time, 10.6 TB/s from
// L2.
constexpr int kLarge = 256;
constexpr int kLargeThreads = 512;
constexpr int kLargeStage = 2 * kLarge * kStage;
constexpr int kLargeLds = 2 * kLargeStage;

__global__ __launch_bounds__(kLargeThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void matmul_large_kernel(
    MatmulArgs a) {
    constexpr int TM = 8, TN = 4, HM = TM / 2, HN = TN / 2;  // blocks of 16 of a wavefront, and of a half of them
    constexpr int kQuarter = 2;                              // loads of a wavefront
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const bool pairs = a.out_type != MI355X_TYPE_F32;
    const int stages = (a.k + kStage - 1) / kStage;
    // a wavefront loads one block of each quarter: of x the row half wave / 4, of w the
    // channels of wavefront wave / 2
    const int x_block = wave / HM * TM + wave % HM, w_block = wave / HN * TN + wave % HN;
    uint32_t x_at[2], w_at[2];
    int chunk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        chunk[i] = piece_chunk(i, lane);
        const int row = piece_row(i, lane);
        x_at[i] = row * static_cast<uint32_t>(a.x_stride) + chunk[i];
        w_at[i] = channel_of(row, 0, pairs) * static_cast<uint32_t>(a.w_stride) + chunk[i];
    }
    const uint32_t x_half = 16 * HM * static_cast<uint32_t>(a.x_stride), w_half = 16 * HN * static_cast<uint32_t>(a.w_stride);
    const int wm = wave & 1, wn = wave >> 1;
    const int x_lds = 2048 * wm * TM, w_lds = 2048 * (16 + wn * TN);
    const int operand[2] = {operand_at(0, col, quad), operand_at(1, col, quad)};
    const int tiles = a.m_tiles * a.n_tiles;

    __amdgpu_buffer_rsrc_t x_rows, w_rows;
    int m0 = 0, n0 = 0;
    // tiles of the last row and column end with the output, over their neighbours' outputs
    auto begin = [&](int t) {
        int mt, nt, split;
        tile_of(a, t, tiles, &mt, &nt, &split);
        m0 = min(mt * kLarge, a.m - kLarge);
        n0 = min(nt * kLarge, a.n - kLarge);
        x_rows = rows_at(a.x + (m0 + 16 * x_block) * a.x_stride);
        w_rows = rows_at(a.w + (n0 + 16 * TN * (wave / HN) + channel_of(0, wave % HN, pairs)) * a.w_stride);
    };
    auto piece = [&](__amdgpu_buffer_rsrc_t rows, uint8_t *dst, const uint32_t *at, uint32_t off, int s) {
        const int k = kStage * s;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t v = at[i];
            if (k + kStage > a.k && k + chunk[i] >= a.k) v -= chunk[i];  // the stage's first
            load_piece(rows, dst + 1024 * i, v, k + off);
        }
    };
    auto load_x = [&](int h, int s) {
        piece(x_rows, lds + (s & 1) * kLargeStage + 2048 * (x_block + h * HM), x_at, h * x_half, s);
    };
    auto load_w = [&](int h, int s) {
        piece(w_rows, lds + (s & 1) * kLargeStage + 2048 * (16 + w_block + h * HN), w_at, h * w_half, s);
    };
    auto load_first = [&]() {
        load_x(0, 0);
        load_w(0, 0);
        load_w(1, 0);
        load_x(1, 0);
        if (stages > 1) {
            load_x(0, 1);
            load_w(0, 1);
            load_w(1, 1);
            load_x(1, 1);
        }
    };
    i32x4 c[TN][TM], x0[2][HM], x1[2][HM], w0[2][HN], w1[2][HN];
    auto read_x = [&](i32x4 (&f)[2][HM], int q, int h, int s) {
#pragma unroll
        for (int j = 0; j < HM; ++j)
            f[q][j] = *reinterpret_cast<const i32x4 *>(lds + (s & 1) * kLargeStage + x_lds + 2048 * (h * HM + j) + operand[q]);
    };
    auto read_w = [&](i32x4 (&f)[2][HN], int h, int s) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < HN; ++i)
                f[q][i] = *reinterpret_cast<const i32x4 *>(lds + (s & 1) * kLargeStage + w_lds + 2048 * (h * HN + i) + operand[q]);
        if (kStage * (s + 1) > a.k)
#pragma unroll
            for (int q = 0; q < 2; ++q)
                if (kStage * s + 64 * q + 16 * quad >= a.k)
#pragma unroll
                    for (int i = 0; i < HN; ++i) f[q][i] = i32x4{0, 0, 0, 0};
    };
    auto multiply = [&](i32x4 (&xf)[2][HM], i32x4 (&wf)[2][HN], int xh, int wh) {
        wait_reads();
        barrier();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < HM; ++j)
#pragma unroll
                for (int i = 0; i < HN; ++i)
                    c[wh * HN + i][xh * HM + j] = mfma(wf[q][i], xf[q][j], c[wh * HN + i][xh * HM + j]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        barrier();
    };
    int t = blockIdx.x;
    if (t >= tiles) return;
    begin(t);
    load_first();
    wait_loads<0>();
    for (;;) {
        // here the first two stages are there for this wavefront's part
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) c[i][j] = i32x4{0, 0, 0, 0};
        barrier();
        if (wave >= 4) barrier();  // the second group is one part behind
        read_x(x0, 0, 0, 0);
        for (int s = 0; s < stages; ++s) {
            const bool more = s + 2 < stages, next = s + 1 < stages;
            read_x(x0, 1, 0, s);
            read_w(w0, 0, s);
            // W1 and X1 of this stage (asked for with it) are there: the next stage's are under way
            if (s >= 2) {
                if (next) wait_loads<4 * kQuarter>();
                else wait_loads<0>();
            }
            multiply(x0, w0, 0, 0);
            read_w(w1, 1, s);
            read_x(x1, 0, 1, s);
            if (more) {
                load_x(0, s + 2);
                load_w(0, s + 2);
            }
            multiply(x0, w1, 0, 1);
            read_x(x1, 1, 1, s);
            // X0 and W0 of the next stage
            if (more) {
                load_w(1, s + 2);
                if (s >= 1) wait_loads<5 * kQuarter>();
            } else if (next && s >= 1) {
                wait_loads<2 * kQuarter>();
            }
            multiply(x1, w1, 1, 1);
            if (next) read_x(x0, 0, 0, s + 1);
            if (more) load_x(1, s + 2);
            multiply(x1, w0, 1, 0);
        }
        if (wave < 4) barrier();  // both groups have read everything
        const int m = m0 + wm * 16 * TM + col, n = n0 + wn * 16 * TN;
        t += gridDim.x;
        const bool last = t >= tiles;
        if (!last) {
            begin(t);
            load_first();
        }
        write_tile<TM, TN>(a, m, n, c, quad, TileScales<TM, TN>(a, m, n, quad));
        if (last) return;
        // of the operations so far only stores of outputs, the newest, may be under way
        if (pairs) wait_loads<TM * TN / 2>();
        else wait_loads<TM * TN>();
    }
}

// ---- launches ------------------------------------------------------------------

constexpr size_t kCounters = size_t(4) * kCounterStep * kMatmulSplitTiles;
constexpr size_t kPartBytes = size_t(kMatmulPartBytes);

template <int TM, int R, int WAVES, int ST>
int launch_few(mi355x_ctx *ctx, const MatmulArgs &a) {
    const dim3 grid((a.n + 16 * R - 1) / (16 * R), (a.m + 16 * TM - 1) / (16 * TM));
    matmul_few_kernel<TM, R, WAVES, ST><<<grid, 64 * WAVES, FewShape<TM, R, WAVES, ST>::kLds, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

// The output in tiles of bm rows and bn channels.
void set_tiles(MatmulArgs &a, int bm, int bn) {
    a.m_tiles = (a.m + bm - 1) / bm;
    a.n_tiles = (a.n + bn - 1) / bn;
    a.tiles = fast_div(static_cast<uint32_t>(a.m_tiles * a.n_tiles));
    a.band = fast_div(static_cast<uint32_t>(8 * a.n_tiles));
    a.last_rows = fast_div(static_cast<uint32_t>(a.m_tiles % 8 ? a.m_tiles % 8 : 8));
}

int stages_of(const MatmulArgs &a) { return (a.k + kStage - 1) / kStage; }

template <int BM, int BN, int WM, int WN, int ST>
int launch_tiles(mi355x_ctx *ctx, MatmulArgs a, int splits) {
    typedef TileShape<BM, BN, WM, WN, ST> S;
    set_tiles(a, BM, BN);
    const int stages = stages_of(a);
    a.split_stages = (stages + splits - 1) / splits;
    a.splits = (stages + a.split_stages - 1) / a.split_stages;
    matmul_tile_kernel<BM, BN, WM, WN, ST>
        <<<static_cast<unsigned>(a.m_tiles * a.n_tiles * a.splits), S::kThreads, S::kLds, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

int launch_large(mi355x_ctx *ctx, MatmulArgs a) {
    set_tiles(a, kLarge, kLarge);
    const int groups = std::min(a.m_tiles * a.n_tiles, ctx->num_cus);
    matmul_large_kernel<<<groups, kLargeThreads, kLargeLds, ctx->stream>>>(a);
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
    const MatmulChoice c = choose_matmul(ctx->num_cus, a.m, a.n, a.k, u.x_stride, u.w_stride);
    switch (c.form) {
    case MatmulForm::kFew16: return launch_few<1, 1, 4, 4>(ctx, a);
    case MatmulForm::kFew16Wide: return launch_few<1, 2, 4, 3>(ctx, a);
    case MatmulForm::kFew32: return launch_few<2, 1, 8, 2>(ctx, a);
    case MatmulForm::kFew32Wide: return launch_few<2, 2, 4, 2>(ctx, a);
    case MatmulForm::kFar: return launch_few<4, 3, 2, 2>(ctx, a);
    case MatmulForm::k64x64: return launch_tiles<64, 64, 4, 2, 4>(ctx, a, c.splits);
    case MatmulForm::k64x128: return launch_tiles<64, 128, 2, 4, 4>(ctx, a, c.splits);
    case MatmulForm::k128x128: return launch_tiles<128, 128, 2, 4, 4>(ctx, a, c.splits);
    case MatmulForm::k256x128: return launch_tiles<256, 128, 2, 4, 3>(ctx, a, c.splits);
    case MatmulForm::k256x256: return launch_large(ctx, a);
    }
    return set_error(MI355X_EINVAL, "mi355x_matmul_q8: no form");
}

}  // namespace mi355x
