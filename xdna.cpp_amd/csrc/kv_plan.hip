// Block tables, slots and positions of a serving step, built on the GPU from
// the requests' lengths.
//
// Two exclusive scans over the requests (new tokens, new pages) give every
// request its rows and its entries of the free list; a row then finds its
// request by a binary search of the offsets.  The work is tens of bytes per
// request and 12 per row, so latency bounds it.
#include "internal.h"
#include "paged_index.h"

#include <algorithm>

namespace mi355x {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Requests whose offsets the one-launch form keeps in LDS.
constexpr int kPlanLdsSeqs = 1024;
// Rows up to which one workgroup writes them itself.
constexpr int64_t kPlanOneLaunchRows = 4096;

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

__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// One workgroup: scans, tables, and (rows) the rows themselves.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(mi355x_kv_plan_args a, int shift, int rows) {
    __shared__ int64_t sums[2][kPlanWaves];
    __shared__ int all_flags;
    __shared__ int32_t off_lds[kPlanLdsSeqs + 1], kv_lds[kPlanLdsSeqs], held_lds[kPlanLdsSeqs], first_lds[kPlanLdsSeqs];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nthr = blockDim.x, nwave = nthr >> 6;
    if (tid == 0) all_flags = 0;
    __syncthreads();
    // totals first: a step that does not fit takes nothing
    int64_t n_new = 0, n_fresh = 0;
    int flags = 0;
    for (int s = tid; s < a.n_seqs; s += nthr) {
        const PlanSeq q = plan_seq(a, shift, s);
        n_new += q.added;
        n_fresh += q.fresh;
        flags |= q.flags;
    }
    n_new = __shfl(wave_scan(n_new, lane), 63);
    n_fresh = __shfl(wave_scan(n_fresh, lane), 63);
    if (flags) atomicOr(&all_flags, flags);
    if (lane == 0) {
        sums[0][wave] = n_new;
        sums[1][wave] = n_fresh;
    }
    __syncthreads();
    n_new = n_fresh = 0;
    for (int w = 0; w < nwave; ++w) {
        n_new += sums[0][w];
        n_fresh += sums[1][w];
    }
    const int64_t head = *a.free_head;
    flags = all_flags;
    if (n_new > a.n_rows) flags |= MI355X_KV_ROWS;
    if (head < 0 || head > a.n_free || n_fresh > a.n_free - head) flags |= MI355X_KV_PAGES;
    __syncthreads();  // every thread has read free_head, which free_head_out may be
    const bool ok = flags == 0;
    if (tid == 0) {
        *a.free_head_out = static_cast<int32_t>(ok ? head + n_fresh : head);
        if (a.status) *a.status = flags;
        a.row_offsets[a.n_seqs] = ok ? static_cast<int32_t>(n_new) : 0;
        if (rows) off_lds[a.n_seqs] = ok ? static_cast<int32_t>(n_new) : 0;
    }
    int64_t carry_new = 0, carry_fresh = 0;
    for (int base = 0; base < a.n_seqs; base += nthr) {
        const int s = base + tid;
        PlanSeq q{};
        if (s < a.n_seqs) q = plan_seq(a, shift, s);
        const int64_t in_new = wave_scan(q.added, lane), in_fresh = wave_scan(q.fresh, lane);
        if (lane == 63) {
            sums[0][wave] = in_new;
            sums[1][wave] = in_fresh;
        }
        __syncthreads();
        int64_t at = carry_new + in_new - q.added, first = head + carry_fresh + in_fresh - q.fresh;
        for (int w = 0; w < nwave; ++w) {
            if (w < wave) {
                at += sums[0][w];
                first += sums[1][w];
            }
            carry_new += sums[0][w];
            carry_fresh += sums[1][w];
        }
        if (s < a.n_seqs) {
            const int64_t kv = ok ? q.cached + q.added : q.cached;
            a.row_offsets[s] = ok ? static_cast<int32_t>(at) : 0;
            a.kv_lens[s] = static_cast<int32_t>(kv);
            if (ok)
                for (int64_t i = 0; i < q.fresh; ++i)
                    a.block_table[s * a.table_stride + q.held + i] = a.free_pages[first + i];
            if (rows) {
                off_lds[s] = ok ? static_cast<int32_t>(at) : 0;
                kv_lds[s] = static_cast<int32_t>(kv);
                held_lds[s] = static_cast<int32_t>(q.held);
                first_lds[s] = static_cast<int32_t>(first);
            }
        }
        __syncthreads();
    }
    if (!rows) return;
    const int64_t real = ok ? n_new : 0;
    for (int64_t r = tid; r < a.n_rows; r += nthr) {
        int32_t pos = 0;
        int64_t slot = -1;
        if (r < real) {
            const int s = seq_of_row(off_lds, a.n_seqs, r);
            pos = static_cast<int32_t>(kv_lds[s] - (off_lds[s + 1] - r));
            const int32_t col = pos >> shift;
            const int32_t page = col < held_lds[s] ? a.block_table[s * a.table_stride + col]
                                                   : a.free_pages[first_lds[s] + (col - held_lds[s])];
            if (page >= 0) slot = (static_cast<int64_t>(page) << shift) + (pos & ((1 << shift) - 1));
        }
        a.positions[r] = pos;
        a.slots[r] = slot;
    }
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
    const bool one = a.n_seqs <= kPlanLdsSeqs && a.n_rows <= kPlanOneLaunchRows;
    const int64_t work = std::max<int64_t>(a.n_seqs, one ? a.n_rows : 0);
    const int threads = static_cast<int>(std::min<int64_t>(kPlanThreads, std::max<int64_t>(64, (work + 63) / 64 * 64)));
    kv_plan_kernel<<<1, threads, 0, ctx->stream>>>(a, shift, one ? 1 : 0);
    MI355X_HIP(hipGetLastError());
    if (!one && a.n_rows > 0) {
        kv_plan_rows_kernel<<<static_cast<unsigned>((a.n_rows + 255) / 256), 256, 0, ctx->stream>>>(a, shift);
        MI355X_HIP(hipGetLastError());
    }
    return MI355X_OK;
}

}  // namespace mi355x
