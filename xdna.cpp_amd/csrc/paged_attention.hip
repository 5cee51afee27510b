// Attention of new tokens over a paged KV cache: the host's choice of form, and
// the token form, for requests that add one or a few tokens.
//
// One pass over a row's keys with the running maximum m and sum l of the
// softmax: a tile of scores s moves m to max(m, s), scales what was summed by
// 2^(m_old - m), and adds 2^(s - m) v and 2^(s - m) (scores carry log2 e).
//
// Token form.  A token reads its whole cache once and does 4 operations per
// value and query head, so HBM bounds it.  The query heads of a KV head (and
// the request's few tokens) are the 16 columns of a matrix product, so that a
// key read once meets all of them: scores as K q^T, one column per row of q, so
// that a lane holds 8 scores of one row of a 32-key tile and the softmax needs
// two exchanges; the weights are then, as they lie, the operand of V^T w, whose
// V^T comes out of LDS through the transposing read.  64 requests of up to 8192
// tokens, 32 query and 8 KV heads of 128: 1.0 GB in 190-197 us, 5.1-5.3 TB/s, as fast as
// a copy; one of 131072 tokens 113 us, 4.8 TB/s.  Short calls are bound by latency:
// lengths, table, keys, parts and their join each wait for the one before (640
// tokens, 2 KV heads: 9.6 us).
//
// Work split.  All requests' keys, heads and row blocks form one line of
// 128-key units; every workgroup takes an equal stretch of it, whatever the
// lengths are, finds its place by a scan over the requests' lengths, and
// writes the output of the rows that lie in its stretch whole.  Of rows that the
// ends of stretches cut each workgroup leaves (m, l, sum) in the workspace, and
// the last of them to get there joins the parts.
#include "attn_device.h"
#include "internal.h"

#include <algorithm>
#include <cfloat>

namespace mi355x {
namespace {

constexpr int kTokenWaves = 4;
constexpr int kTokenKeys = 32;                            // of a wavefront's tile
constexpr int kUnitKeys = kTokenWaves * kTokenKeys;       // of a workgroup's unit
constexpr int kTokenThreads = 64 * kTokenWaves;
constexpr int kTokenRows = 16;                            // head rows of a workgroup: columns of a product

// The token form's units of a request: per KV head and block of kTokenRows head rows
// one per kUnitKeys keys (one without keys: its rows get zeros).
struct TokenWork {
    int64_t units;
    int blocks, tiles, key_lo;
};

__device__ __forceinline__ TokenWork token_work(const AttnArgs &a, const SeqGeo &g) {
    TokenWork w{0, 0, 1, 0};
    if (g.rows <= 0 || g.rows > a.row_limit) return w;
    w.blocks = (g.rows + kTokenRows - 1) / kTokenRows;
    w.key_lo = token_keys(a, g, g.tok_lo).lo;
    w.tiles = max(1, (token_keys(a, g, g.tok_lo + g.n_tok - 1).hi - w.key_lo + kUnitKeys - 1) / kUnitKeys);
    w.units = static_cast<int64_t>(w.blocks) * w.tiles * a.n_kv_heads;
    return w;
}

// The units before each request, a request per thread.  Up to 64 requests: every
// wavefront scans them by itself (one request of 640 tokens 9.8 us against 10.1, 64
// ragged ones 194 against 196).  More: the workgroup does, all of them at once or a
// part at a time.
template <int WAVES>
struct Scan {
    int64_t total;
    int64_t mine, before;  // of request threadIdx.x (% 64)
    int32_t row_begin, row_end, kv;  // up to 64 requests: its offsets and length

    // Request s's rows and tokens, which up to 64 requests' lanes have.
    __device__ __forceinline__ SeqGeo geo(const AttnArgs &a, int s) const {
        if (a.n_seqs > 64) return seq_geo(a, s);
        return seq_geo(a, __builtin_amdgcn_readlane(row_begin, s), __builtin_amdgcn_readlane(row_end, s),
                       __builtin_amdgcn_readlane(kv, s));
    }

    __device__ __forceinline__ void run(const AttnArgs &a, int64_t *tmp) {
        if (a.n_seqs <= 64) {
            const int lane = threadIdx.x & 63;
            row_begin = row_end = kv = 0;
            if (lane < a.n_seqs) {
                row_begin = a.row_offsets[lane];
                row_end = a.row_offsets[lane + 1];
                kv = a.kv_lens[lane];
            }
            mine = lane < a.n_seqs ? token_work(a, seq_geo(a, row_begin, row_end, kv)).units : 0;
            int64_t in = mine;
            if (a.n_seqs > 1)
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int64_t u = __shfl_up(in, d);
                    if (lane >= d) in += u;
                }
            before = in - mine;
            total = uniform(__shfl(in, a.n_seqs - 1));
            return;
        }
        total = 0;
        for (int base = 0; base < a.n_seqs; base += 64 * WAVES) {
            const int s = base + threadIdx.x;
            const int64_t n = s < a.n_seqs ? token_work(a, seq_geo(a, s)).units : 0;
            int64_t sum;
            const int64_t at = group_scan<WAVES>(n, tmp, &sum);
            if (base == 0) {
                mine = n;
                before = at;
            }
            total += sum;
        }
        total = uniform(total);
    }

    // The request that has unit u < total, and the units before it.
    __device__ __forceinline__ int find(const AttnArgs &a, int64_t u, int64_t *tmp, int64_t *first) const {
        if (a.n_seqs <= 64) {
            const uint64_t here = __ballot(u >= before && u < before + mine);
            const int s = __builtin_ctzll(here | (uint64_t(1) << 63));
            *first = uniform(__shfl(before, s));
            return s;
        }
        int64_t n = mine, at = before, carry = 0;
        __shared__ int64_t found_at;
        __shared__ int found;
        for (int base = 0; base < a.n_seqs; base += 64 * WAVES) {
            const int s = base + threadIdx.x;
            if (a.n_seqs > 64 * WAVES) {
                int64_t sum;
                n = s < a.n_seqs ? token_work(a, seq_geo(a, s)).units : 0;
                at = carry + group_scan<WAVES>(n, tmp, &sum);
                carry += sum;
            }
            if (u >= at && u < at + n) {
                found = s;
                found_at = at;
            }
        }
        __syncthreads();
        *first = uniform(found_at);
        const int s = __builtin_amdgcn_readfirstlane(found);
        __syncthreads();
        return s;
    }
};

// How the units are shared out.  A stretch of u units takes about u steps, and the
// join of N / u parts, eight of which each of its teams loads at a time, N / (8 u
// teams) and more: u = sqrt(N / (12 teams)) of the average N, where there are
// workgroups to spare (16 heads of 128, 2 KV heads: one request of 16000 tokens 21
// us, 26 with a unit each; of 64000 31, 54; 4 of 5000 14.9, 18.0).
__device__ __forceinline__ Stretches token_line(const AttnArgs &a, int64_t total) {
    const float wanted = sqrtf(static_cast<float>(total) * a.line_share) + 0.5f;
    int64_t groups = gridDim.x;
    if (wanted >= 2.0f) {
        const int64_t u = static_cast<int64_t>(wanted);
        groups = idx_min(groups, quotient(total + u - 1, u));
    }
    return stretches(total, static_cast<int>(groups));
}

template <int HD>
struct TokenShape {
    static constexpr int kVStride = HD + 16;  // values: rows of V start 8 banks apart
    static constexpr int kWaveBytes = kTokenKeys * kVStride * 2;
    static constexpr int kOStride = HD + 4;   // floats of a joined row
    static_assert(16 * kOStride * 4 <= kWaveBytes, "a wavefront's sums fit where its V tile was");
    // a part in the workspace: sums of kTokenRows rows, then m, then l
    static constexpr int kPartFloats = kTokenRows * (HD + 2);
};

template <int TYPE, int HD, int PLANES>
__global__ __launch_bounds__(kTokenThreads, HD <= 64 ? 3 : HD <= 128 ? 2 : 1) void attention_token_kernel(AttnArgs a) {
    typedef Num<TYPE> N;
    typedef typename N::T T;
    typedef typename N::V8 V8;
    typedef TokenShape<HD> S;
    constexpr int kSteps = HD / 32;     // of a 16-key score product
    constexpr int kBlocks = HD / 16;    // of 16 output values
    constexpr int kChunks = HD / 8;     // 16-byte chunks of a token's head
    constexpr int kVLoads = kTokenKeys * kChunks / 64;
    __shared__ __attribute__((aligned(16))) unsigned char lds[kTokenWaves * S::kWaveBytes];
    __shared__ float lds_m[kTokenWaves][16], lds_l[kTokenWaves][16];
    __shared__ int lds_odd[kTokenWaves];
    __shared__ int64_t tmp[kTokenWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    Scan<kTokenWaves> scan;
    scan.run(a, tmp);
    const Stretches line = token_line(a, scan.total);
    if (static_cast<int>(blockIdx.x) >= line.groups) return;
    const int64_t u0 = stretch_begin(line, blockIdx.x), u1 = stretch_begin(line, blockIdx.x + 1);
    if (u0 >= u1) return;
    int64_t before;  // units before request seq
    int seq = scan.find(a, u0, tmp, &before);
    T *vt = reinterpret_cast<T *>(lds + wave * S::kWaveBytes);
    float *ot = reinterpret_cast<float *>(lds + wave * S::kWaveBytes);
    SeqGeo g = scan.geo(a, seq);
    TokenWork w = token_work(a, g);
    for (int64_t u = u0; u < u1;) {
        while (u >= before + w.units) {  // the next request with rows
            before += w.units;
            ++seq;
            g = scan.geo(a, seq);
            w = token_work(a, g);
        }
        const int64_t item = quotient(u - before, w.tiles);
        const int t0 = static_cast<int>(u - before - item * w.tiles);
        const int t1 = static_cast<int>(idx_min(w.tiles, t0 + (u1 - u)));
        const int kvh = static_cast<int>(quotient(item, w.blocks));
        const int row0 = static_cast<int>(item - static_cast<int64_t>(kvh) * w.blocks) * kTokenRows;
        const int row_last = min(row0 + kTokenRows, g.rows) - 1;
        // tokens that some row of the block sees, and those that all of them see
        const Keys kf = token_keys(a, g, g.tok_lo + divided(row0, a.group));
        const Keys kl = token_keys(a, g, g.tok_lo + divided(row_last, a.group));
        const int all_lo = kl.lo, all_hi = kf.hi;
        const bool whole = t0 == 0 && t1 == w.tiles;

        V8 qf[kSteps];
        const bool real = row0 + col < g.rows;
        const int row = real ? row0 + col : 0, tok = divided(row, a.group);
        const Keys mine = token_keys(a, g, g.tok_lo + tok);
        const int row_lo = mine.lo, row_hi = real ? mine.hi : 0;
        {
            const int64_t head = static_cast<int64_t>(kvh) * a.group.d + (row - tok * static_cast<int>(a.group.d));
            const T *q = static_cast<const T *>(a.q) + (g.first + g.tok_lo + tok) * a.q_stride + head * HD;
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                V8 z = {};
                if (real) z = *reinterpret_cast<const V8 *>(q + 32 * st + 8 * quad);
                qf[st] = z;
            }
        }
        const int32_t *table = a.table + seq * a.table_stride;
        const T *kp = static_cast<const T *>(a.k) + kvh * a.head_stride + 8 * quad;
        const T *vp = static_cast<const T *>(a.v) + kvh * a.head_stride;

        // Tokens [some_lo, some_hi) are seen by some row; the others' values count as
        // zero.  Where a value that only some of the rows see is not finite (a weight of
        // zero would not take it away), the rows are done again one by one.
        int some_lo = kf.lo, some_hi = kl.hi;
        bool odd = false;
        for (int only = -1; only < kTokenRows; ++only) {
            if (only >= 0) {
                if (!odd || row0 + only >= g.rows) break;
                const Keys kr = token_keys(a, g, g.tok_lo + divided(row0 + only, a.group));
                some_lo = kr.lo;
                some_hi = kr.hi;
            }
            bool odd_lane = false;
            f32x4 o[kBlocks];
            Reference<TYPE> ref;
            float l = 0.0f;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) o[d] = f32x4{0, 0, 0, 0};

            u32x4_a kreg[2][kSteps], vreg[kVLoads];
            uint32_t seen = 0;  // keys of the tile in registers that lie on pages of the pool
            // the table entry of key (lane & 31) of a tile
            auto entry = [&](int base) {
                const int key = base + (lane & 31);
                return key >= some_lo && key < some_hi ? table[key >> a.shift] : -1;
            };
            auto load = [&](int base, int32_t page) {
                const bool good = page_in_pool(page, a.n_pages);
                const int64_t off = good ? token_at(a, page, base + (lane & 31)) : 0;
                seen = static_cast<uint32_t>(__ballot(good));
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const T *k = kp + __shfl(off, 16 * b + col);
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) kreg[b][st] = *reinterpret_cast<const u32x4_a *>(k + 32 * st);
                }
#pragma unroll
                for (int i = 0; i < kVLoads; ++i) {
                    const int idx = 64 * i + lane;
                    const T *v = vp + __shfl(off, idx / kChunks) + idx % kChunks * 8;
                    vreg[i] = *reinterpret_cast<const u32x4_a *>(v);
                }
            };
            // this wavefront's tiles: every kTokenWaves-th
            const int first = w.key_lo + t0 * kUnitKeys + wave * kTokenKeys;
            const int end = min(some_hi, w.key_lo + t1 * kUnitKeys);
            int32_t next = -1;
            if (first < end) {
                load(first, entry(first));
                next = entry(first + kUnitKeys);
            }
            for (int base = first; base < end; base += kUnitKeys) {
                const uint32_t now = seen;
                float s[8];  // keys 16 (i / 4) + 4 quad + i % 4
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    f32x4 c = {0, 0, 0, 0};
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) c = N::mfma16(__builtin_bit_cast(V8, kreg[b][st]), qf[st], c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[4 * b + i] = c[i];
                }
                // every key of the tile seen by every row
                const bool full = base >= all_lo && base + kTokenKeys <= all_hi && now == 0xFFFFFFFFu;
#pragma unroll
                for (int i = 0; i < kVLoads; ++i) {
                    const int idx = 64 * i + lane, key = idx / kChunks;
                    u32x4_a v = vreg[i];
                    if (!full) {
                        if (!((now >> key) & 1)) v = u32x4_a{0, 0, 0, 0};
                        odd_lane |= not_finite<TYPE>(v);
                    }
                    *reinterpret_cast<u32x4_a *>(vt + key * S::kVStride + idx % kChunks * 8) = v;
                }
                const int after = base + kUnitKeys;
                if (after < end) {
                    load(after, next);
                    next = entry(after + kUnitKeys);
                }
                scores2(s, a);
                if (!full) {
                    const uint32_t see = (now & range_mask<uint32_t>(row_lo, row_hi, base)) >> (4 * quad);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!((see >> (16 * (i >> 2) + (i & 3))) & 1)) s[i] = -INFINITY;
                }
                float top = s[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
                top = quad_max(top);
                const bool moves = ref.moves(top);
                const float keep = ref.move(moves, top);
                if (__any(moves)) {
                    l *= keep;
#pragma unroll
                    for (int d = 0; d < kBlocks; ++d) o[d] *= keep;
                }
                const float zero = ref.base();
                V8 w[PLANES];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = __builtin_amdgcn_exp2f(s[i] - zero);
                    l += p;
                    split_weight<TYPE, PLANES>(p, w, i);
                }
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) {
                    const T *p = vt + (4 * quad + col / 4) * S::kVStride + 16 * d + col % 4 * 4;
                    const u32x2_a x = lds_read_transposed(reinterpret_cast<const s16x4 *>(p)),
                                  y = lds_read_transposed(reinterpret_cast<const s16x4 *>(p + 16 * S::kVStride));
                    const V8 v = __builtin_bit_cast(V8, u32x4_a{x[0], x[1], y[0], y[1]});
#pragma unroll
                    for (int i = 0; i < PLANES; ++i) o[d] = N::mfma16(v, w[i], o[d]);
                }
            }

            // join the wavefronts' sums
            const FarParts parts(a.ws);
            const int part = (2 * blockIdx.x + (u != u0)) * S::kPartFloats;
            const float sum = quad_sum(l);
            if (quad == 0) {
                lds_m[wave][col] = ref.m;
                lds_l[wave][col] = sum;
            }
            if (only < 0) {
                const bool any = __any(odd_lane);
                if (lane == 0) lds_odd[wave] = any;
            }
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
                *reinterpret_cast<f32x4 *>(ot + col * S::kOStride + 16 * d + 4 * quad) = o[d];
            __syncthreads();
            if (only < 0)
                for (int wv = 0; wv < kTokenWaves; ++wv) odd |= lds_odd[wv] != 0;
            int start = tid;
            asm volatile("" : "+v"(start));  // the addresses below are formed here, not kept through the loops
            for (int idx = start; idx < kTokenRows * (HD / 4); idx += kTokenThreads) {
                const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
                if (row0 + r >= g.rows) break;
                if (only >= 0 && r != only) continue;
                Joined j;
#pragma unroll
                for (int wv = 0; wv < kTokenWaves; ++wv)
                    j.add(lds_m[wv][r], lds_l[wv][r],
                          *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(lds + wv * S::kWaveBytes) +
                                                           r * S::kOStride + c));
                if (whole) {
                    store_out4<TYPE>(a, out_at(a, g, kvh, row0 + r, HD) + c, j.value());
                } else {
                    parts.store4(part + r * HD + c, j.num);
                    if (c == 0) {
                        parts.store(part + kTokenRows * HD + r, j.top);
                        parts.store(part + kTokenRows * (HD + 1) + r, j.den);
                    }
                }
            }
            __syncthreads();
        }
        if (!whole) {
            const int64_t begin = u - t0, end = begin + w.tiles;
            const int64_t from = stretch_of(line, begin);
            const int n_parts = static_cast<int>(stretch_of(line, end - 1) - from) + 1;
            if (last_of(a.counters + from, n_parts, &lds_odd[0])) {
                // the first part ends its stretch (unless it is all of it), the others begin theirs
                const FarParts parts(a.ws);
                const int second = begin != stretch_begin(line, from);
                auto part_of = [&](int i) {
                    return (2 * (static_cast<int>(from) + i) + (i == 0 ? second : 0)) * S::kPartFloats;
                };
                // a thread per row and 4 values, and as many teams of them as fit share the parts
                constexpr int kQuads = HD / 4;
                f32x4 *nums = reinterpret_cast<f32x4 *>(lds);
                float *dens = reinterpret_cast<float *>(nums + kTokenThreads), *tops = dens + kTokenThreads;
                const int rows = row_last - row0 + 1;
                int id = tid;
                asm volatile("" : "+v"(id));  // as above
                for (int r0 = 0; r0 < rows; r0 += kTokenThreads / kQuads) {
                    const int n = min(kTokenThreads / kQuads, rows - r0) * kQuads;
                    const int teams = min(n_parts, kTokenThreads / n), team = id / n;
                    const int r = r0 + id % n / kQuads, c = id % kQuads * 4;
                    Joined j;
                    if (team < teams)
                        join_parts(
                            j, parts, n_parts, team, teams, [&](int i) { return part_of(i) + r * HD + c; },
                            [&](int i) { return part_of(i) + kTokenRows * HD + r; },
                            [&](int i) { return part_of(i) + kTokenRows * (HD + 1) + r; });
                    nums[id] = j.num;
                    dens[id] = j.den;
                    tops[id] = j.top;
                    __syncthreads();
                    if (team == 0) {
                        for (int t = 1; t < teams; ++t) j.add(tops[t * n + id], dens[t * n + id], nums[t * n + id]);
                        store_out4<TYPE>(a, out_at(a, g, kvh, row0 + r, HD) + c, j.value());
                    }
                    __syncthreads();
                }
            }
            __syncthreads();  // lds_odd, lds
        }
        u += t1 - t0;
    }
}

// The token form runs as many workgroups as stay on the chip together.
constexpr int kTokenGroupsPerCu = 4;

template <int TYPE, int HD, int PLANES>
int launch_planes(mi355x_ctx *ctx, const AttnArgs &a) {
    const void *kernel = reinterpret_cast<const void *>(attention_token_kernel<TYPE, HD, PLANES>);
    const int64_t fit = ctx->num_cus * std::max(1, std::min(kTokenGroupsPerCu, occupancy(kernel, kTokenThreads, 0)));
    // no more than the units that the table allows
    const int64_t heads = static_cast<int64_t>(a.n_seqs) * a.n_kv_heads;
    const int64_t units = heads * (a.reach / kUnitKeys + 1);
    attention_token_kernel<TYPE, HD, PLANES>
        <<<static_cast<unsigned>(std::min(fit, units)), kTokenThreads, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

template <int TYPE, int HD>
int launch_token(mi355x_ctx *ctx, const AttnArgs &a) {
    return a.f32_out ? launch_planes<TYPE, HD, f32_planes(TYPE)>(ctx, a) : launch_planes<TYPE, HD, 2>(ctx, a);
}

// rows: the host's bound on a request's head rows.  Up to kTokenRows the token
// form; else the chunk form, behind the token form for the requests that add
// few (one request alone takes the chunk form at once).  With more rows the token form
// reads the keys again for every kTokenRows of them; the chunk form is as fast or
// faster from 17 on (us, chunk form against token form; contexts of 500 to 6000
// tokens): 16 requests of 5 tokens and 8 heads 29.7, 38.0; of 5 and 4 71.6, 85.4; of 8
// and 4 71.7, 87.1; of 17 and 1 70.9, 85.5; of 1 and 32 21.9, 21.8; 64 of 3 tokens and 8
// heads 71.8, 84.7, of 16 and 4 214, 672; one of 4 and 8 on 30000 tokens 32.8, 33.2.
template <int TYPE, int HD>
int launch_forms(mi355x_ctx *ctx, const AttnArgs &a, int64_t rows) {
    if (rows <= kTokenRows) return launch_token<TYPE, HD>(ctx, a);
    AttnArgs b = a;
    b.row_limit = 0;
    if (a.n_seqs > 1) {
        AttnArgs c = a;
        c.row_limit = b.row_limit = kTokenRows;
        if (int rc = launch_token<TYPE, HD>(ctx, c)) return rc;
    }
    return launch_attention_chunk(ctx, b, TYPE, HD);
}

template <int TYPE>
int launch_sizes(mi355x_ctx *ctx, const AttnArgs &a, int head_dim, int64_t rows) {
    switch (head_dim) {
    case 64: return launch_forms<TYPE, 64>(ctx, a, rows);
    case 96: return launch_forms<TYPE, 96>(ctx, a, rows);
    case 128: return launch_forms<TYPE, 128>(ctx, a, rows);
    default: return launch_forms<TYPE, 256>(ctx, a, rows);
    }
}

}  // namespace

// One counter per workgroup of the token form.
static size_t counter_bytes(const mi355x_ctx *ctx) {
    return (static_cast<size_t>(ctx->num_cus) * kTokenGroupsPerCu * 4 + 255) / 256 * 256;
}

size_t paged_attention_workspace_bytes(const mi355x_ctx *ctx, int, int, int head_dim) {
    return counter_bytes(ctx) + std::max(static_cast<size_t>(ctx->num_cus * kTokenGroupsPerCu) * 2 * kTokenRows * (head_dim + 2) * 4,
                                         attention_chunk_workspace(ctx, head_dim));
}

int launch_paged_attention(mi355x_ctx *ctx, const mi355x_paged_attention_args &u) {
    AttnArgs a{};
    a.q = u.q;
    a.k = u.pool->k;
    a.v = u.pool->v;
    a.row_offsets = u.row_offsets;
    a.kv_lens = u.kv_lens;
    a.table = u.block_table;
    a.out = u.out;
    a.counters = static_cast<int *>(u.workspace);
    a.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(u.workspace) + counter_bytes(ctx));
    a.q_stride = u.q_stride;
    a.out_stride = u.out_stride;
    a.table_stride = u.table_stride;
    a.page_stride = static_cast<uint32_t>(u.pool->page_stride);
    a.token_stride = static_cast<uint32_t>(u.pool->token_stride);
    a.head_stride = u.pool->head_stride;
    a.n_rows = u.n_rows;
    // an empty pool has no address that may be read: no token is seen
    a.reach = u.pool->n_pages > 0 ? u.table_cols * u.pool->page_tokens : 0;
    a.scale2 = u.scale * kLog2e;
    if (u.softcap > 0.0f) {
        a.cap_in = std::max(-FLT_MAX, std::min(FLT_MAX, u.scale / u.softcap * (2.0f * kLog2e)));
        a.cap_out = u.softcap * kLog2e;
    }
    a.n_seqs = u.n_seqs;
    a.n_kv_heads = u.pool->n_kv_heads;
    const int group = u.n_heads / u.pool->n_kv_heads;
    a.group = fast_div(static_cast<uint32_t>(group));
    a.n_pages = static_cast<int>(u.pool->n_pages);
    a.shift = __builtin_ctz(static_cast<unsigned>(u.pool->page_tokens));
    a.window = u.window;
    a.causal = u.causal;
    a.row_limit = INT32_MAX;
    const int64_t added = u.max_added > 0 ? std::min<int64_t>(u.max_added, u.n_rows) : u.n_rows;
    const int join_threads = static_cast<int>(std::min<int64_t>(kTokenRows, added * group)) * (u.pool->head_dim / 4);
    a.line_share = 1.0f / (12.0f * static_cast<float>(std::max(1, kTokenThreads / join_threads)) *
                           static_cast<float>(u.n_seqs) * static_cast<float>(u.pool->n_kv_heads));
    a.f32_out = u.out_type == MI355X_TYPE_F32;
    return u.pool->type == MI355X_TYPE_F16
               ? launch_sizes<MI355X_TYPE_F16>(ctx, a, u.pool->head_dim, added * group)
               : launch_sizes<MI355X_TYPE_BF16>(ctx, a, u.pool->head_dim, added * group);
}

}  // namespace mi355x
