// Which kernel a product of 8-bit integers takes, and in how many parts of k: host
// arithmetic alone, shared with the CPU tests (no HIP in here).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace mi355x {

constexpr int kMatmulStage = 128;                       // bytes of k in a stage
constexpr int kMatmulSplitTiles = 1024;                 // tiles whose k may be split: each has a counter
constexpr int64_t kMatmulPartBytes = int64_t(64) << 20; // room for all parts' sums

// Few rows, up to 16 or 32, a workgroup 16 or (wide) 32 channels; rows far apart; tiles of
// rows x channels.
enum class MatmulForm { kFew16, kFew16Wide, kFew32, kFew32Wide, kFar, k64x64, k64x128, k128x128, k256x128, k256x256 };
struct MatmulChoice {
    MatmulForm form;
    int splits;
};

// Tiles, the time that a workgroup takes for a stage of k where it has a CU for itself
// and where `per_cu` share one (of one row of tiles: weights come from memory, and not
// from an L2), and what the first and each later round of workgroups takes besides (us).
struct MatmulTiles {
    MatmulForm form;
    int bm, bn, per_cu, most_splits;
    float alone, shared, alone_one_row, shared_one_row, first, later;
};
constexpr MatmulTiles kMatmulTiles[] = {
    {MatmulForm::k64x64, 64, 64, 2, 8, 0.29f, 0.53f, 0.31f, 0.65f, 0.5f, 0.5f},
    {MatmulForm::k64x128, 64, 128, 1, 8, 0.47f, 0.47f, 0.57f, 0.57f, 0.5f, 0.5f},
    {MatmulForm::k128x128, 128, 128, 1, 8, 0.66f, 0.66f, 0.66f, 0.66f, 0.5f, 2.5f},
    {MatmulForm::k256x128, 256, 128, 1, 8, 0.96f, 0.96f, 0.96f, 0.96f, 0.5f, 7.0f},
    {MatmulForm::k256x256, 256, 256, 1, 1, 1.60f, 1.60f, 1.60f, 1.60f, 6.4f, 6.4f},
};

// The tiles and the split of k with the least estimated time: the launch, rounds of
// workgroups, and for a split the parts that a tile's last workgroup reads; operands
// come from memory at 4.4 TB/s at most.  us measured, weights taken in turn from 1 GB of
// them so that none waits in a cache, of the forms in order with their best split in
// parentheses: 37 x 17408, k 5120: 28 (2), 26.6 (1).  64 x 28672, k 4096: 30
// (1), 30 (1).  64 x 2048, k 11008: 12.7 (6), 15 (8).  201 x 2560, k 2048: 8 (1), 9 (1), 12 (3),
// 17 (2).  200 x 22016, k 2048: 31, 30, 28, 22 (1).  300 x 5120, k 5120: 26 (1), 23 (1), 21 (2),
// 30 (2), 64.  256 x 8192, k 8192: 39 (1), 33 (1), 31 (2), 36 (4), 92.  512 x 4096, k 14336:
// 63 (1), 52 (1), 44 (2), 46 (4), 154.  1024 x 4096, k 4096: 37, 33, 25 (1), 31 (2), 51.  512 x
// 22016, k 2048: 54, 59, 43, 43, 33.  5000 x 5000, k 2048: 105, 106, 85, 82, 65.  Of these the
// least is chosen in each, and elsewhere one within 10% of the least.
inline MatmulChoice choose_matmul_tiles(int num_cus, int m, int n, int k) {
    const int stages = (k + kMatmulStage - 1) / kMatmulStage;
    const float from_memory = static_cast<float>(m + n) * static_cast<float>(k) / 4.4e6f;
    MatmulChoice best{MatmulForm::k64x64, 1};
    float least = 1e30f;
    for (const MatmulTiles &g : kMatmulTiles) {
        // (the large tiles end with the output, and so do not leave it)
        if (g.form == MatmulForm::k256x256 && (m < g.bm || n < g.bn)) continue;
        const int64_t tiles = static_cast<int64_t>((m + g.bm - 1) / g.bm) * ((n + g.bn - 1) / g.bn);
        const int64_t tile_bytes = int64_t(4) * g.bm * g.bn;
        for (int s = 1; s <= g.most_splits && s <= stages; ++s) {
            const int64_t groups = tiles * s;
            // (parts in more than one round did not gain: 37 x 17408, k 5120 in 5 parts 31 us, whole 27)
            if (s > 1 && (groups > num_cus * g.per_cu || tiles > kMatmulSplitTiles || groups * tile_bytes > kMatmulPartBytes))
                break;
            const float rounds = std::ceil(static_cast<float>(groups) / static_cast<float>(num_cus * g.per_cu));
            const bool alone = groups <= num_cus, one_row = m <= g.bm;
            float us = (rounds - 1.0f) * g.later +
                       rounds * (one_row ? alone ? g.alone_one_row : g.shared_one_row : alone ? g.alone : g.shared) *
                           static_cast<float>((stages + s - 1) / s);
            if (s > 1) us += 1.5f + static_cast<float>(s) * static_cast<float>(tile_bytes) / 32768.0f;
            us = 3.2f + g.first + std::max(us, from_memory);
            if (us < least) {
                least = us;
                best = {g.form, s};
            }
        }
    }
    return best;
}

inline MatmulChoice choose_matmul(int num_cus, int m, int n, int k, int64_t x_stride, int64_t w_stride) {
    // the tile kernels form offsets of up to 256 rows in 32 bits
    const bool far = x_stride > (1 << 23) || w_stride > (1 << 23);
    // Up to 32 rows have the weight in flight in each wavefront by itself; blocks of 32
    // channels where that fills the CUs, else of 16 so that more workgroups share the work
    // (16, then 32 channels; us, weights from memory as above: one row of 2048, k 11008 7.6, 10.4;
    // of 8192, k 8192 12.9, 12.9; of 22016, k 2048 11.6, 10.1; 32 rows of 2048, k 2048 3.5, 4.0; of
    // 22016 20, 12).  The tiles take more: 32 rows of 2048, k 2048 7.0, of 22016 13.9; 17 of 28672,
    // k 4096 27.6, here 24.5; 37 rows 28.6, here (48 channels, 48 rows) 31.3.
    const bool many = n >= 32 * num_cus;
    if (m <= 16) return {many ? MatmulForm::kFew16Wide : MatmulForm::kFew16, 1};
    if (m <= 32) return {many ? MatmulForm::kFew32Wide : MatmulForm::kFew32, 1};
    if (far) return {MatmulForm::kFar, 1};
    return choose_matmul_tiles(num_cus, m, n, k);
}

}  // namespace mi355x
