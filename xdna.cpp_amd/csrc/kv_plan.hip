// Block tables, slots and positions of a serving step, built on the GPU from
// the requests' lengths.
//
// Sums over the requests (new tokens, new pages) give every request its rows and
// its entries of the free list; a row then finds its request by a binary search of
// the offsets.  The work is tens of bytes per
// request and 12 per row, so latency bounds it.
#include "internal.h"
#include "paged_index.h"

#include <algorithm>

namespace mi355x {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Requests up to which one launch does it all, a request per thread.
constexpr int kPlanOneLaunchSeqs = kPlanThreads;
// Rows up to which one workgroup writes those of a step in place (64 requests, from
// call to result: 1 row each 13 us against 18 with a second launch for the rows,
// 4096 rows 18 against 20).
constexpr int64_t kPlanInPlaceRows = 4096;

struct PlanSeq {
    int64_t cached, added, held, fresh;
    int flags;
};

__device__ __forceinline__ PlanSeq plan_seq(const mi355x_kv_plan_args &a, int shift, int s) {
    PlanSeq q;
    q.cached = a.cached[s];
    q.added = a.added[s];
    q.flags = q.cached < 0 || q.added < 0 || q.cached + q.added > INT32_MAX ? MI355X_KV_BAD_LENGTH : 0;
    if (q.flags) {
        q.cached = idx_max(q.cached, 0);
        q.added = q.held = q.fresh = 0;
        return q;
    }
    q.held = pages_of(q.cached, shift);
    const int64_t need = pages_of(q.cached + q.added, shift);
    q.fresh = need - q.held;
    if (need > a.table_cols) q.flags |= MI355X_KV_TABLE;
    return q;
}

// Inclusive sums over a wavefront, held at 2^32 - 1: a total of 2^31 or more does
// not fit anyway, and then no sum is used.
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ uint32_t sum_step(uint32_t v) {
    const uint32_t u = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROW_MASK, 0xF, false);
    return __builtin_elementwise_add_sat(v, u);
}
__device__ __forceinline__ uint32_t wave_sums(uint32_t v) {
    v = sum_step<0x111>(v);       // row_shr:1
    v = sum_step<0x112>(v);       // row_shr:2
    v = sum_step<0x114>(v);       // row_shr:4
    v = sum_step<0x118>(v);       // row_shr:8
    v = sum_step<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    return sum_step<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// The sums before this thread's values over the workgroup, and the totals.
struct PlanSums {
    uint32_t rows, pages, all_rows, all_pages;
};
__device__ __forceinline__ PlanSums group_sums(uint32_t rows, uint32_t pages, uint32_t (*tmp)[kPlanWaves]) {
    const int wave = threadIdx.x >> 6, n = blockDim.x >> 6;
    const uint32_t in_rows = wave_sums(rows), in_pages = wave_sums(pages);
    if ((threadIdx.x & 63) == 63) {
        tmp[0][wave] = in_rows;
        tmp[1][wave] = in_pages;
    }
    __syncthreads();
    PlanSums s{in_rows - rows, in_pages - pages, 0, 0};
    for (int w = 0; w < n; ++w) {
        if (w < wave) {
            s.rows = __builtin_elementwise_add_sat(s.rows, tmp[0][w]);
            s.pages = __builtin_elementwise_add_sat(s.pages, tmp[1][w]);
        }
        s.all_rows = __builtin_elementwise_add_sat(s.all_rows, tmp[0][w]);
        s.all_pages = __builtin_elementwise_add_sat(s.all_pages, tmp[1][w]);
    }
    return s;
}

__device__ __forceinline__ int plan_flags(const mi355x_kv_plan_args &a, int flags, const PlanSums &s, int64_t head) {
    if (s.all_rows > a.n_rows) flags |= MI355X_KV_ROWS;
    if (head < 0 || head > a.n_free || s.all_pages > a.n_free - head) flags |= MI355X_KV_PAGES;
    return flags;
}

// What belongs to request s but its table, and what belongs to the step.
__device__ __forceinline__ void write_seq(const mi355x_kv_plan_args &a, int s, const PlanSeq &q, int64_t row, bool ok) {
    a.row_offsets[s] = ok ? static_cast<int32_t>(row) : 0;
    a.kv_lens[s] = static_cast<int32_t>(ok ? q.cached + q.added : q.cached);
}
__device__ __forceinline__ void write_step(const mi355x_kv_plan_args &a, int64_t rows, int64_t head, int flags) {
    a.row_offsets[a.n_seqs] = static_cast<int32_t>(rows);
    *a.free_head_out = static_cast<int32_t>(head);
    if (a.status) *a.status = flags;
}

// Up to kPlanOneLaunchSeqs requests: sums, tables and rows in one launch.  Each of
// several workgroups takes a part of the rows and sums over all requests for
// itself, which costs less than a second launch (65 thousand rows of 256 requests
// 4.7 us against 9.4); the first one writes what belongs to the requests.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(mi355x_kv_plan_args a, int shift, int group_rows) {
    __shared__ uint32_t sums[2][kPlanWaves];
    __shared__ int all_flags;
    __shared__ int32_t off[kPlanOneLaunchSeqs + 1], kv_len[kPlanOneLaunchSeqs], held[kPlanOneLaunchSeqs],
        fresh_at[kPlanOneLaunchSeqs];
    const int tid = threadIdx.x, nthr = blockDim.x;
    const int64_t head = *a.free_head;
    PlanSeq q{};
    if (tid < a.n_seqs) q = plan_seq(a, shift, tid);
    if (tid == 0) all_flags = 0;
    __syncthreads();
    if (q.flags) atomicOr(&all_flags, q.flags);
    const PlanSums s = group_sums(static_cast<uint32_t>(q.added), static_cast<uint32_t>(q.fresh), sums);
    // every thread of a workgroup has read what the first one may write in place
    const int flags = plan_flags(a, all_flags, s, head);
    const bool ok = flags == 0;
    const int64_t rows = ok ? s.all_rows : 0;
    if (blockIdx.x == 0) {
        if (tid < a.n_seqs) write_seq(a, tid, q, s.rows, ok);
        if (tid == 0) write_step(a, rows, ok ? head + s.all_pages : head, flags);
    }
    if (tid < a.n_seqs) {
        off[tid] = ok ? static_cast<int32_t>(s.rows) : 0;
        kv_len[tid] = static_cast<int32_t>(q.cached + q.added);
        held[tid] = static_cast<int32_t>(q.held);
        fresh_at[tid] = static_cast<int32_t>(head + s.pages);
    }
    if (tid == 0) off[a.n_seqs] = static_cast<int32_t>(rows);
    __syncthreads();
    const int64_t row_end = idx_min(a.n_rows, (static_cast<int64_t>(blockIdx.x) + 1) * group_rows);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * group_rows + tid; r < row_end; r += nthr) {
        int32_t pos = 0;
        int64_t slot = -1;
        if (r < rows) {
            const int t = seq_of_row(off, a.n_seqs, r);
            pos = static_cast<int32_t>(kv_len[t] - (off[t + 1] - r));
            const int32_t col = pos >> shift;
            // an entry that stands, or a new one, which its page's first row writes
            int32_t *entry = a.block_table + t * a.table_stride + col;
            int32_t page;
            if (col < held[t]) {
                page = *entry;
            } else {
                page = a.free_pages[fresh_at[t] + (col - held[t])];
                if ((pos & ((1 << shift) - 1)) == 0) *entry = page;
            }
            if (page >= 0) slot = (static_cast<int64_t>(page) << shift) + (pos & ((1 << shift) - 1));
        }
        a.positions[r] = pos;
        a.slots[r] = slot;
    }
}

// More requests: one workgroup sums, a part of the requests at a time.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_seqs_kernel(mi355x_kv_plan_args a, int shift) {
    __shared__ uint32_t sums[2][kPlanWaves];
    __shared__ int all_flags;
    __shared__ int32_t fresh_at[kPlanThreads + 1], held[kPlanThreads];
    const int tid = threadIdx.x;
    const int64_t head = *a.free_head;
    if (tid == 0) all_flags = 0;
    PlanSums all{};
    // totals first: a step that does not fit takes nothing
    for (int base = 0; base < a.n_seqs; base += kPlanThreads) {
        __syncthreads();
        PlanSeq q{};
        if (base + tid < a.n_seqs) q = plan_seq(a, shift, base + tid);
        if (q.flags) atomicOr(&all_flags, q.flags);
        const PlanSums s = group_sums(static_cast<uint32_t>(q.added), static_cast<uint32_t>(q.fresh), sums);
        all.all_rows = __builtin_elementwise_add_sat(all.all_rows, s.all_rows);
        all.all_pages = __builtin_elementwise_add_sat(all.all_pages, s.all_pages);
    }
    __syncthreads();
    const int flags = plan_flags(a, all_flags, all, head);
    const bool ok = flags == 0;
    uint32_t rows = 0, pages = 0;
    for (int base = 0; base < a.n_seqs; base += kPlanThreads) {
        __syncthreads();
        PlanSeq q{};
        if (base + tid < a.n_seqs) q = plan_seq(a, shift, base + tid);
        const PlanSums s = group_sums(static_cast<uint32_t>(q.added), static_cast<uint32_t>(q.fresh), sums);
        if (base + tid < a.n_seqs) write_seq(a, base + tid, q, int64_t(rows) + s.rows, ok);
        if (ok) {
            // the part's new pages, side by side in the free list, a thread each
            fresh_at[tid] = static_cast<int32_t>(s.pages);
            held[tid] = static_cast<int32_t>(q.held);
            if (tid == 0) fresh_at[kPlanThreads] = static_cast<int32_t>(s.all_pages);
            __syncthreads();
            for (int64_t i = tid; i < s.all_pages; i += kPlanThreads) {
                const int t = seq_of_row(fresh_at, kPlanThreads, i);
                a.block_table[(base + t) * a.table_stride + held[t] + (i - fresh_at[t])] = a.free_pages[head + pages + i];
            }
        }
        rows = __builtin_elementwise_add_sat(rows, s.all_rows);
        pages = __builtin_elementwise_add_sat(pages, s.all_pages);
    }
    if (tid == 0) write_step(a, ok ? all.all_rows : 0, ok ? head + all.all_pages : head, flags);
}

// Rows of a step whose offsets, lengths and tables stand already.
__global__ __launch_bounds__(256) void kv_plan_rows_kernel(mi355x_kv_plan_args a, int shift) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= a.n_rows) return;
    int32_t pos = 0;
    int64_t slot = -1;
    const int s = seq_of_row(a.row_offsets, a.n_seqs, r);
    if (s >= 0) {
        pos = static_cast<int32_t>(a.kv_lens[s] - (a.row_offsets[s + 1] - r));
        const int32_t page = a.block_table[s * a.table_stride + (pos >> shift)];
        if (page >= 0) slot = (static_cast<int64_t>(page) << shift) + (pos & ((1 << shift) - 1));
    }
    a.positions[r] = pos;
    a.slots[r] = slot;
}

}  // namespace

int launch_kv_plan(mi355x_ctx *ctx, const mi355x_kv_plan_args &a) {
    const int shift = __builtin_ctz(static_cast<unsigned>(a.page_tokens));
    // several workgroups may not read what the first one writes in place
    const bool in_place = a.kv_lens == a.cached || a.free_head_out == a.free_head;
    // a request per thread, and threads for the rows: of a small step, or of one in
    // place (4096 rows: 26 us from call to result with 256, 18 with 1024)
    const int64_t most = std::max<int64_t>(a.n_seqs, std::min<int64_t>(a.n_rows, in_place ? kPlanThreads : 256));
    const int threads = static_cast<int>(std::min<int64_t>(kPlanThreads, std::max<int64_t>(64, (most + 63) / 64 * 64)));
    if (a.n_seqs <= kPlanOneLaunchSeqs && (!in_place || a.n_rows <= kPlanInPlaceRows)) {
        const int64_t groups = in_place ? 1 : std::max<int64_t>(1, std::min<int64_t>(1024, (a.n_rows + threads - 1) / threads));
        const int64_t rows = (std::max<int64_t>(a.n_rows, 1) + groups - 1) / groups;
        kv_plan_kernel<<<static_cast<unsigned>(groups), threads, 0, ctx->stream>>>(a, shift, static_cast<int>(rows));
        MI355X_HIP(hipGetLastError());
        return MI355X_OK;
    }
    kv_plan_seqs_kernel<<<1, kPlanThreads, 0, ctx->stream>>>(a, shift);
    MI355X_HIP(hipGetLastError());
    if (a.n_rows > 0) {
        kv_plan_rows_kernel<<<static_cast<unsigned>((a.n_rows + 255) / 256), 256, 0, ctx->stream>>>(a, shift);
        MI355X_HIP(hipGetLastError());
    }
    return MI355X_OK;
}

}  // namespace mi355x
