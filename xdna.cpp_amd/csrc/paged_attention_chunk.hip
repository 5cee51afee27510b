// Attention over a paged KV cache, chunk form: for requests that add many
// tokens.
//
// A workgroup takes 128 or 256 head rows (tokens x query heads of one KV head) of a
// request and walks the keys that they see in tiles of 64; a wavefront owns 32
// of the rows.  As in the token form a tile's scores are K q^T, so that a lane
// holds 32 scores of one row, the softmax needs one exchange, and the weights
// are, as they lie, the operand of V^T w; O^T stays in registers.  Matrix cores and
// vector units bound it, one after the other: a prompt of 8192 tokens, 32 query and 8 KV
// heads of 128, is 0.55 Tflop at 540-608 us, 0.9-1.0 Pflop/s, with the matrix cores
// busy in 43% of the cycles and vector instructions in 47%, where products of 8192 x
// 8192 matrices reach 1.39 on the card with 69% and 10%.  Without its exponentials
// it takes 40 us less, without its loads 48, with a quarter of the second product 115;
// neither priorities nor products between the exponentials move it.
//
// K and V tiles travel to LDS directly (global_load_lds), one tile ahead.  Such
// loads fill LDS in lane order, so rows cannot be padded; instead the 16-byte
// chunks of a row are permuted by the row's number (the lane that fills a place
// loads the chunk that belongs there), so that neither the score operands (32
// rows, one chunk) nor the transposed reads of V (4 rows, two chunks) meet in a
// bank (counted: none).
//
// Work split.  Blocks of rows are numbered so that a workgroup finds its
// request from the row offsets alone; the last ones (which see the most keys)
// start first.  Where they leave CUs idle the keys of each are cut into `split`
// parts, which leave (m, l, sum) in the workspace for a second launch.
#include "attn_device.h"
#include "internal.h"

#include <algorithm>

namespace mi355x {
namespace {

constexpr int kChunkKeys = 64;
// Softcaps (times log2 e) up to which 1 - 2 / (1 + e^2y) is near enough to tanh y, to
// 2^-23 of the cap (24 mixed requests, cap 30: 60 us; with the series below 1/8, 75).
constexpr float kNearCap = 64.0f;
// Instruction kinds of __builtin_amdgcn_sched_group_barrier.
constexpr int kMfma = 0x8, kDsRead = 0x100;

template <int HD, int WAVES>
struct ChunkShape {
    static constexpr int kThreads = 64 * WAVES;
    static constexpr int kRows = 32 * WAVES;
    static constexpr int kChunks = HD / 8;                            // 16-byte chunks of a token's head
    static constexpr int kPlaces = HD == 96 ? 16 : kChunks;           // places for them in LDS, a power of two
    static constexpr int kRowBytes = 16 * kPlaces;
    static constexpr int kTileBytes = kChunkKeys * kRowBytes;
    static constexpr int kLoads = kChunkKeys * kPlaces / kThreads;  // of K, and of V, per lane
    static constexpr int kPartFloats = kRows * (HD + 2);
    static constexpr int kLds = 4 * kTileBytes;                       // K and V, two tiles each
};

// The place of chunk c of row r is c ^ turn: 16 consecutive rows' chunk c (K), or
// 4 chunks of 4 consecutive rows (V), lie in the 16 places that make up LDS's 64
// banks.  (Rows of 32 places: 8 of them for K, so that a lane fills the same
// chunk of all its rows.)
template <int PLACES>
__device__ __forceinline__ int k_turn(int r) {
    return PLACES == 8 ? (r >> 1) & 7 : PLACES == 16 ? r & 15 : r & 7;
}
template <int PLACES>
__device__ __forceinline__ int v_turn(int r) {
    return PLACES == 8 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
}

// The request whose blocks of 2^SHIFT rows include block j, its first one, and its
// rows and tokens.  Up to 64 requests: a lane has loaded what belongs to each, so
// that no load waits for the search.
template <int SHIFT>
__device__ __forceinline__ int find_block(const AttnArgs &a, int64_t j, int64_t *first, SeqGeo *g) {
    // ascends by at least 1: one block more at every seam
    auto begin = [&](int32_t offset, int s) { return ((static_cast<int64_t>(offset) * a.group.d) >> SHIFT) + s; };
    const int lane = threadIdx.x & 63;
    if (a.n_seqs <= 64) {
        const int s = min(lane, a.n_seqs - 1);
        const int32_t from = a.row_offsets[s], to = a.row_offsets[s + 1], kv = a.kv_lens[s];
        const uint64_t below = __ballot(lane < a.n_seqs && begin(from, s) <= j);
        const int found = 63 - __builtin_clzll(below | 1);
        const int32_t offset = __builtin_amdgcn_readlane(from, found);
        *first = begin(offset, found);
        *g = seq_geo(a, offset, __builtin_amdgcn_readlane(to, found), __builtin_amdgcn_readlane(kv, found));
        return found;
    }
    int lo = 0, n = a.n_seqs;  // the request is in lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) / 64;
        const int s = lo + lane * step;
        const uint64_t below = __ballot(lane * step < n && begin(a.row_offsets[s], s) <= j);
        const int k = max(0, 63 - __builtin_clzll(below | 1));
        n = min(step, n - k * step);
        lo += k * step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    *g = seq_geo(a, lo);
    *first = begin(a.row_offsets[lo], lo);
    return lo;
}

struct ChunkItem {
    int seq, kvh, row0;
    SeqGeo g;
    Keys first, last;  // of the block's first and last row
    int tiles;         // of keys from key_lo on
    int key_lo;
};

constexpr int row_shift(int waves) { return waves == 8 ? 8 : 7; }

// False: no rows there.
template <int WAVES>
__device__ __forceinline__ bool chunk_item(const AttnArgs &a, int64_t j, int kvh, ChunkItem *it) {
    int64_t begin;
    constexpr int kRows = 32 * WAVES;
    static_assert(kRows == 1 << row_shift(WAVES), "blocks of rows");
    it->seq = find_block<row_shift(WAVES)>(a, j, &begin, &it->g);
    it->kvh = kvh;
    const int64_t row0 = (j - begin) * kRows;
    if (row0 < 0 || row0 >= it->g.rows || it->g.rows <= a.row_limit) return false;
    it->row0 = static_cast<int>(row0);
    const int row_last = min(it->row0 + kRows, it->g.rows) - 1;
    it->first = token_keys(a, it->g, it->g.tok_lo + divided(it->row0, a.group));
    it->last = token_keys(a, it->g, it->g.tok_lo + divided(row_last, a.group));
    it->key_lo = it->first.lo & ~(kChunkKeys - 1);
    it->tiles = (max(it->last.hi - it->key_lo, 0) + kChunkKeys - 1) / kChunkKeys;
    return true;
}

template <int TYPE, int HD, bool CAP, int PLANES, int WAVES>
__global__ __launch_bounds__(64 * WAVES, HD > 128 ? 1 : 2) void attention_chunk_kernel(AttnArgs a) {
    typedef Num<TYPE> N;
    typedef typename N::T T;
    typedef typename N::V8 V8;
    typedef ChunkShape<HD, WAVES> S;
    constexpr int kThreads = S::kThreads, kRows = S::kRows;
    constexpr int kSteps = HD / 16;   // of a 32-key score product
    constexpr int kBlocks = HD / 32;  // of 32 output values
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    __shared__ int odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    // block = ((j from the last on) * split + part) * KV heads + head
    const int kvh = static_cast<int>(blockIdx.x % a.n_kv_heads);
    const int64_t rest = blockIdx.x / a.n_kv_heads;
    const int part = static_cast<int>(rest % a.split);
    ChunkItem it;
    if (!chunk_item<WAVES>(a, gridDim.x / (a.n_kv_heads * a.split) - 1 - rest / a.split, kvh, &it)) return;
    const SeqGeo g = it.g;
    const int t0 = static_cast<int>(static_cast<int64_t>(it.tiles) * part / a.split);
    const int t1 = static_cast<int>(static_cast<int64_t>(it.tiles) * (part + 1) / a.split);

    // this lane's row
    const int row_raw = it.row0 + 32 * wave + col;
    const bool real = row_raw < g.rows;
    const int row = real ? row_raw : 0, tok = divided(row, a.group), group = static_cast<int>(a.group.d);
    const int64_t head = static_cast<int64_t>(kvh) * group + (row - tok * group);
    const Keys mine = token_keys(a, g, g.tok_lo + tok);
    const int row_lo = mine.lo, row_hi = real ? mine.hi : 0;
    V8 qf[kSteps];
    {
        const T *q = static_cast<const T *>(a.q) + (g.first + g.tok_lo + tok) * a.q_stride + head * HD;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            V8 z = {};
            if (real) z = *reinterpret_cast<const V8 *>(q + 16 * st + 8 * half);
            qf[st] = z;
        }
    }
    // where this lane's loads come from: its chunk of a token's head (the turn of the
    // rows that it fills is the same), and where it reads: K row
    // col (+ 32), chunk 2 st + half; V rows 4 half + (lane % 16) / 4 (+ 8 ..), chunk
    // 4 d + 2 ((lane / 16) % 2) + (lane % 4) / 2
    const int fill_row = (wave * 64 + lane) / S::kPlaces;
    static_assert(kThreads / S::kPlaces % (S::kPlaces == 32 ? 8 : 16) == 0, "one turn for all of a lane's rows");
    int ck = lane % S::kPlaces ^ k_turn<S::kPlaces>(fill_row), cv = lane % S::kPlaces ^ v_turn<S::kPlaces>(fill_row);
    if (HD == 96) {  // places without a chunk take another's
        ck = ck < S::kChunks ? ck : ck - 4;
        cv = cv < S::kChunks ? cv : cv - 4;
    }
    // a wavefront's load covers kFillRows consecutive rows; where those share a page
    // (a.by_page) its address is one scalar and an offset per lane (prompt of 8192
    // tokens 8 us of 556)
    constexpr int kFillRows = 64 / S::kPlaces, kFillStep = kThreads / S::kPlaces;
    const T *kp = static_cast<const T *>(a.k) + kvh * a.head_stride, *vp = static_cast<const T *>(a.v) + kvh * a.head_stride;
    const uint32_t k_off = 2 * ((lane / S::kPlaces) * a.token_stride + 8 * ck);  // bytes
    const uint32_t v_off = 2 * ((lane / S::kPlaces) * a.token_stride + 8 * cv);
    const int k_at = col * S::kRowBytes;
    const int k_low = half ^ k_turn<S::kPlaces>(col);
    const int v_row = 4 * half + ((lane & 15) >> 2);
    const int v_at = v_row * S::kRowBytes + (lane & 1) * 8;
    const int v_low = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_turn<S::kPlaces>(v_row);
    const int32_t *table = a.table + it.seq * a.table_stride;
    // A row's scores are c1 y + c0, c1 > 0, of the values y that the loop below keeps
    // and compares: of q . k, of -1 / (1 + e^2y) under a cap (a weight then costs one
    // operation less), or of the scores themselves.
    const bool near_cap = CAP && a.cap_out > 0.0f && a.cap_out <= kNearCap;
    const float c1 = CAP ? near_cap ? 2.0f * a.cap_out : 1.0f : a.scale2, c0 = near_cap ? a.cap_out : 0.0f;

    // Tokens [some_lo, some_hi) are seen by some row; the others' values count as
    // zero.  Where a value that only some of the rows see is not finite (a weight of
    // zero would not take it away), the rows are done again one by one.
    int some_lo = it.first.lo, some_hi = it.last.hi;
    if (tid == 0) odd = 0;
    for (int only = -1; only < kRows; ++only) {
        if (only >= 0) {
            __syncthreads();
            if (odd == 0 || it.row0 + only >= g.rows) break;
            const Keys kr = token_keys(a, g, g.tok_lo + divided(it.row0 + only, a.group));
            some_lo = kr.lo;
            some_hi = kr.hi;
        }
        f32x16 o[kBlocks];
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
        Reference<TYPE> ref;
        float l = 0.0f;
        const int col_lo = some_lo >> a.shift, col_hi = (some_hi - 1) >> a.shift;
        // the table entry of key `lane` of tile t, if some row sees a token on its page
        auto entry = [&](int t) {
            const int column = (it.key_lo + t * kChunkKeys + lane) >> a.shift;
            return t < t1 && column >= col_lo && column <= col_hi ? table[column] : -1;
        };
        uint64_t seen_next = 0;  // keys of the tile on its way that some row sees, on pages of the pool
        auto load = [&](int t, int32_t entry, int buf) {
            const bool good = page_in_pool(entry, a.n_pages);
            const int base = it.key_lo + t * kChunkKeys, page = good ? entry : 0;
            seen_next = __ballot(good) & range_mask<uint64_t>(some_lo, some_hi, base);
            unsigned char *to = lds + 2 * buf * S::kTileBytes + 1024 * wave;
            // the load's first row: kFillRows wave + kFillStep i
            if (a.by_page) {
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) {
                    const int row = kFillRows * wave + i * kFillStep;
                    const int64_t from = token_at(a, __builtin_amdgcn_readlane(page, row), base + row);
                    load_lds16(reinterpret_cast<const char *>(kp + from) + k_off, to + 16 * kThreads * i);
                    load_lds16(reinterpret_cast<const char *>(vp + from) + v_off,
                               to + S::kTileBytes + 16 * kThreads * i);
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < S::kLoads; ++i) {
                    const int row = kFillRows * wave + i * kFillStep + lane / S::kPlaces;
                    const int64_t from = token_at(a, __shfl(page, row), base + row);
                    load_lds16(kp + from + 8 * ck, to + 16 * kThreads * i);
                    load_lds16(vp + from + 8 * cv, to + S::kTileBytes + 16 * kThreads * i);
                }
            }
        };
        int32_t next = -1;
        if (t0 < t1) {
            load(t0, entry(t0), 0);
            next = entry(t0 + 1);
        }
        for (int t = t0; t < t1; ++t) {
            const int buf = (t - t0) & 1;
            const uint64_t seen = seen_next;
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this tile's loads
            __syncthreads();                     // everyone's, and the other buffer is read
            if (t + 1 < t1) {
                load(t + 1, next, buf ^ 1);
                next = entry(t + 2);
            }
            unsigned char *kt = lds + 2 * buf * S::kTileBytes, *vt = kt + S::kTileBytes;
            const int base = it.key_lo + t * kChunkKeys;
            // every key of the tile seen by every row of the workgroup
            const bool full = base >= it.last.lo && base + kChunkKeys <= it.first.hi && ~seen == 0;
            if (!full) {
                bool bad = false;
                for (int i = tid; i < kChunkKeys * S::kPlaces; i += kThreads) {
                    u32x4_a *p = reinterpret_cast<u32x4_a *>(vt + 16 * i);
                    if (!((seen >> (i / S::kPlaces)) & 1)) *p = u32x4_a{0, 0, 0, 0};
                    else bad |= not_finite<TYPE>(*p);
                }
                if (__any(bad) && lane == 0) odd = 1;
                __syncthreads();
            }
            // keys that no row of this wavefront sees (heads of 256: one wavefront on a SIMD, where
            // skipping frees nothing, and without it the sums' registers need no copies: 512
            // tokens on 4096 73 us against 78, 4096 tokens of 4 heads 195 against 203, with a
            // cap 197 against 280)
            if (HD <= 128 && !__any(row_lo < base + kChunkKeys && row_hi > base)) continue;
            float s[32];  // keys 32 (i / 16) + 8 (i / 4 % 4) + 4 half + i % 4
            f32x16 x[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[0][i] = x[1][i] = 0.0f;
#pragma unroll
            for (int st = 0; st < kSteps; ++st)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const int place = (2 * st) ^ k_low;
                    const V8 k = *reinterpret_cast<const V8 *>(kt + k_at + 32 * kb * S::kRowBytes + 16 * place);
                    x[kb] = N::mfma32(k, qf[st], x[kb]);
                }
            // operands kAhead reads ahead of their products: left alone, each waits for its own
            constexpr int kAhead = 6;
            __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
            for (int i = 0; i < 2 * kSteps - kAhead; ++i) {
                __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kMfma, kAhead, 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = x[0][i];
                s[16 + i] = x[1][i];
            }
            if (near_cap) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[i] * a.cap_in));
            } else if (CAP) {
                scores2(s, a);
            }
            // every key seen by every row of this wavefront
            if (!full && !__all(row_lo <= base && base + kChunkKeys <= row_hi && ~seen == 0)) {
                const uint64_t see = (seen & range_mask<uint64_t>(row_lo, row_hi, base)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!((see >> (32 * (i >> 4) + 8 * ((i >> 2) & 3) + (i & 3))) & 1)) s[i] = -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i]);
            top = half_max(top);
            top = fmaf(top, c1, c0);
            const bool moves = ref.moves(top);
            if (__any(moves)) {
                const float keep = ref.move(moves, top);
                l *= keep;
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) o[d] *= keep;
            }
            const float base2 = c0 - ref.base();
            auto v_chunk = [&](int j, int d) {  // keys 16 j + {4 half .. + 3, 8 + 4 half .. + 3} of 32 values
                const int place = (4 * d) ^ v_low;
                const s16x4 *p = reinterpret_cast<const s16x4 *>(vt + v_at + 16 * j * S::kRowBytes + 16 * place);
                const u32x2_a x = lds_read_transposed(p), y = lds_read_transposed(p + S::kRowBytes);
                return __builtin_bit_cast(V8, u32x4_a{x[0], x[1], y[0], y[1]});
            };
            // the next 16 keys' reads go out before this 16 keys' weights are formed (the
            // fences keep that order: left alone, each product waits for its own read)
            V8 v[2][kBlocks];
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) v[0][d] = v_chunk(0, d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < 3)
#pragma unroll
                    for (int d = 0; d < kBlocks; ++d) v[(j + 1) & 1][d] = v_chunk(j + 1, d);
                __builtin_amdgcn_sched_barrier(0);
                V8 w[PLANES];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = s[8 * j + i], p = __builtin_amdgcn_exp2f(fmaf(y, c1, base2));
                    l += p;
                    split_weight<TYPE, PLANES>(p, w, i);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                    for (int i = 0; i < PLANES; ++i) o[d] = N::mfma32(v[j & 1][d], w[i], o[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        l = half_sum(l);
        int r = 32 * wave + col;
        asm volatile("" : "+v"(r));  // the addresses below are formed here, not kept through the loops
        if (real && (only < 0 || r == only)) {
            if (a.split == 1) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int64_t at = out_at(a, g, kvh, it.row0 + r, HD);
#pragma unroll
                for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 v = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                        store_out4<TYPE>(a, at + 32 * d + 8 * i + 4 * half, l == 0.0f ? f32x4{0, 0, 0, 0} : v * inv);
                    }
            } else {
                float *w = a.ws + static_cast<int64_t>(blockIdx.x) * S::kPartFloats;
#pragma unroll
                for (int d = 0; d < kBlocks; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4 *>(w + r * HD + 32 * d + 8 * i + 4 * half) =
                            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                if (half == 0) {
                    w[kRows * HD + r] = ref.m;
                    w[kRows * (HD + 1) + r] = l;
                }
            }
        }
    }
}

// Joins the parts of each row block and KV head: a workgroup kJoinRows of its
// rows, a thread 4 values.  (In the kernel above, by the last of a block's
// workgroups, the parts of a chunk of 512 tokens cost 40 us instead of 7.6: one CU
// reads what 16 do here.)
constexpr int kJoinThreads = 256;

template <int TYPE, int HD, int WAVES>
__global__ __launch_bounds__(kJoinThreads) void attention_chunk_join_kernel(AttnArgs a) {
    typedef ChunkShape<HD, WAVES> S;
    constexpr int kRows = S::kRows, kQuads = HD / 4;
    const int kvh = static_cast<int>(blockIdx.x % a.n_kv_heads);
    const int rest = static_cast<int>(blockIdx.x / a.n_kv_heads), blocks = static_cast<int>(gridDim.x / a.n_kv_heads);
    ChunkItem it;
    if (!chunk_item<WAVES>(a, blocks - 1 - rest, kvh, &it)) return;
    const int i = threadIdx.x + kJoinThreads * blockIdx.y, r = i / kQuads, c = i % kQuads * 4;
    if (r >= kRows || r >= it.g.rows - it.row0) return;
    Joined j;
    auto part_of = [&](int p) { return ((rest * a.split + p) * a.n_kv_heads + kvh) * S::kPartFloats; };
    join_parts(
        j, NearParts(a.ws), a.split, 0, 1, [&](int p) { return part_of(p) + r * HD + c; },
        [&](int p) { return part_of(p) + kRows * HD + r; }, [&](int p) { return part_of(p) + kRows * (HD + 1) + r; });
    store_out4<TYPE>(a, out_at(a, it.g, kvh, it.row0 + r, HD) + c, j.value());
}

// Blocks of 2^shift rows as find_block numbers them: request s begins at
// floor(offset_s / 2^shift) + s and takes ceil(rows_s / 2^shift) of them, so the
// last one ends at ceil(rows / 2^shift) + n_seqs - 1 at most.
int64_t row_blocks(int64_t rows, int shift, int n_seqs) {
    return ((rows + (int64_t(1) << shift) - 1) >> shift) + n_seqs - 1;
}

// Workgroups that a call is split into at most, while that is more than its row blocks:
// as many as run at once (heads of 256: one on a CU; 512 tokens on 4096 73 us, 87
// with twice as many).
template <int HD, int WAVES>
int chunk_groups(const mi355x_ctx *ctx) { return (HD > 128 ? 1 : 8 / WAVES) * ctx->num_cus; }

template <int TYPE, int HD, bool CAP, int PLANES, int WAVES>
int launch_blocks(mi355x_ctx *ctx, AttnArgs a) {
    const int64_t items = row_blocks(a.n_rows * a.group.d, row_shift(WAVES), a.n_seqs) * a.n_kv_heads;
    // few blocks: parts of their keys, for the tiles of all CUs (a chunk of 512 tokens on
    // 4096, 64 blocks: 46 us, 141 unsplit; 53 with half as many again), of no fewer than
    // four tiles where the table allows that many tokens
    a.split = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>(chunk_groups<HD, WAVES>(ctx) / items, (int64_t(a.reach) + 4 * kChunkKeys - 1) / (4 * kChunkKeys))));
    attention_chunk_kernel<TYPE, HD, CAP, PLANES, WAVES>
        <<<static_cast<unsigned>(items * a.split), 64 * WAVES, ChunkShape<HD, WAVES>::kLds, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    if (a.split > 1) {
        const dim3 grid(static_cast<unsigned>(items), (32 * WAVES * HD / 4 + kJoinThreads - 1) / kJoinThreads);
        attention_chunk_join_kernel<TYPE, HD, WAVES><<<grid, kJoinThreads, 0, ctx->stream>>>(a);
        MI355X_HIP(hipGetLastError());
    }
    return MI355X_OK;
}

// Workgroups of 256 rows load half as much into LDS per row, but a request's last
// one leaves more wavefronts without rows: they are for requests of 2048 rows and
// more on average (us with 128 -> 256 rows: a prompt of 8192 tokens and 4 heads 586
// -> 556; one request of 4096 rows 46.2 -> 43.8, 8 of them 81 -> 76; 8 of 2048 70 ->
// 68; one of 1024 20.7 -> 23.2; 64 of 132 129 -> 153, of 800 407 -> 426).  Heads of 64
// values leave registers for three workgroups of 128 rows on a CU (4096 tokens
// and 4 heads 96 us, 101 with 256 rows), heads of 256 none for 256 rows.
template <int TYPE, int HD, bool CAP, int PLANES>
int launch_chunk(mi355x_ctx *ctx, const AttnArgs &args) {
    AttnArgs a = args;
    a.by_page = a.shift >= __builtin_ctz(64 / ChunkShape<HD, 4>::kPlaces) && a.token_stride < (1u << 26);
    if constexpr (HD == 96 || HD == 128)
        if (a.n_rows * a.group.d >= 2048 * int64_t(a.n_seqs)) return launch_blocks<TYPE, HD, CAP, PLANES, 8>(ctx, a);
    return launch_blocks<TYPE, HD, CAP, PLANES, 4>(ctx, a);
}

template <int TYPE, int HD>
int launch_size(mi355x_ctx *ctx, const AttnArgs &a) {
    // the common path masks and takes the maximum before it scales, for which the scale has to be positive
    const bool cap = a.cap_out > 0.0f || !(a.scale2 > 0.0f);
    constexpr int kPlanes = f32_planes(TYPE);
    if (a.f32_out)
        return cap ? launch_chunk<TYPE, HD, true, kPlanes>(ctx, a) : launch_chunk<TYPE, HD, false, kPlanes>(ctx, a);
    return cap ? launch_chunk<TYPE, HD, true, 1>(ctx, a) : launch_chunk<TYPE, HD, false, 1>(ctx, a);
}

template <int TYPE>
int launch_type(mi355x_ctx *ctx, const AttnArgs &a, int head_dim) {
    switch (head_dim) {
    case 64: return launch_size<TYPE, 64>(ctx, a);
    case 96: return launch_size<TYPE, 96>(ctx, a);
    case 128: return launch_size<TYPE, 128>(ctx, a);
    default: return launch_size<TYPE, 256>(ctx, a);
    }
}

}  // namespace

size_t attention_chunk_workspace(const mi355x_ctx *ctx, int head_dim) {
    // the same floats for workgroups of 128 and of 256 rows
    const int groups = head_dim > 128 ? chunk_groups<256, 4>(ctx) : chunk_groups<128, 4>(ctx);
    return static_cast<size_t>(groups) * 128 * (head_dim + 2) * 4;
}

int launch_attention_chunk(mi355x_ctx *ctx, const AttnArgs &a, int type, int head_dim) {
    return type == MI355X_TYPE_F16 ? launch_type<MI355X_TYPE_F16>(ctx, a, head_dim)
                                   : launch_type<MI355X_TYPE_BF16>(ctx, a, head_dim);
}

}  // namespace mi355x
