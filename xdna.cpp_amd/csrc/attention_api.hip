// Entry points of mi355x-attention.h: what the host can check of a call's
// arguments, the device gate, and the launch.
#include "internal.h"
#include "mi355x-attention.h"

#include <climits>
#include <cmath>
#include <string>

namespace mi355x {
namespace {

constexpr int kMostSeqs = 65536;
constexpr int kMostPageTokens = 65536;

int invalid(const char *who, const std::string &what) {
    return set_error(MI355X_EINVAL, std::string(who) + ": " + what);
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int type_bytes(int type) {
    return type == MI355X_TYPE_F32 ? 4 : type == MI355X_TYPE_F16 || type == MI355X_TYPE_BF16 ? 2 : 0;
}

int check_page_tokens(const char *who, int n) {
    if (n < 1 || n > kMostPageTokens || (n & (n - 1)) != 0)
        return invalid(who, "page_tokens must be a power of two up to 65536 (got " + std::to_string(n) + ")");
    return MI355X_OK;
}

// Offsets inside the pool are formed in 64 bits: page * page_stride and the
// rest must not overflow.
int check_pool(const char *who, const mi355x_kv_pool *p) {
    if (p->type != MI355X_TYPE_F16 && p->type != MI355X_TYPE_BF16)
        return invalid(who, "the pool's type must be F16 or BF16 (got " + std::to_string(p->type) + ")");
    if (p->n_kv_heads < 1) return invalid(who, "the pool needs at least one head");
    if (p->head_dim < 8 || p->head_dim % 8 != 0)
        return invalid(who, "the pool's head_dim must be a multiple of 8 (got " + std::to_string(p->head_dim) + ")");
    if (int rc = check_page_tokens(who, p->page_tokens)) return rc;
    if (p->n_pages < 0 || p->n_pages > INT32_MAX)
        return invalid(who, "n_pages must be 0 to 2^31 - 1 (got " + std::to_string(p->n_pages) + ")");
    if (p->n_pages > 0 && (!p->k || !p->v)) return invalid(who, "null pool");
    if (!aligned(p->k, 16) || !aligned(p->v, 16)) return invalid(who, "the pool must be 16-byte aligned");
    constexpr int64_t kMostStride = int64_t(1) << 31;  // the kernels form products of 32-bit numbers
    for (int64_t s : {p->page_stride, p->token_stride, p->head_stride})
        if (s < 0 || s % 8 != 0 || s > kMostStride)
            return invalid(who, "pool strides must be multiples of 8 values, 0 to 2^31 (got " + std::to_string(s) + ")");
    return MI355X_OK;
}

int check_rows(const char *who, int64_t n) {
    if (n < 0 || n > INT32_MAX) return invalid(who, "n_rows must be 0 to 2^31 - 1 (got " + std::to_string(n) + ")");
    return MI355X_OK;
}

int check_seqs(const char *who, int n) {
    if (n < 0 || n > kMostSeqs) return invalid(who, "n_seqs must be 0 to 65536 (got " + std::to_string(n) + ")");
    return MI355X_OK;
}

// A row of `heads` heads and the stride between rows, for n rows.
int check_row_stride(const char *who, const char *name, int64_t n, int64_t stride, int64_t width) {
    if (stride < 0 || stride > (int64_t(1) << 40) || (n > 1 && stride < width))
        return invalid(who, std::string(name) + " must be at least a row's " + std::to_string(width) +
                                " values and at most 2^40 (got " + std::to_string(stride) + ")");
    return MI355X_OK;
}

}  // namespace
}  // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_kv_plan(mi355x_ctx *ctx, const mi355x_kv_plan_args *args) {
    clear_error();
    static const char *who = "mi355x_kv_plan";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_kv_plan_args &a = *args;
    if (int rc = check_seqs(who, a.n_seqs)) return rc;
    if (int rc = check_page_tokens(who, a.page_tokens)) return rc;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (a.table_cols < 0 || a.n_free < 0) return invalid(who, "negative table_cols or n_free");
    if (a.table_stride < 0 || a.table_stride > INT32_MAX || (a.n_seqs > 1 && a.table_stride < a.table_cols))
        return invalid(who, "table_stride must be at least table_cols and at most 2^31 - 1 (got " +
                                std::to_string(a.table_stride) + ")");
    if (!a.free_head || !a.free_head_out || !a.row_offsets) return invalid(who, "null pointer argument provided");
    if (a.n_seqs > 0 && (!a.cached || !a.added || !a.kv_lens)) return invalid(who, "null pointer argument provided");
    if (a.n_seqs > 0 && a.table_cols > 0 && !a.block_table) return invalid(who, "null block_table");
    if (a.n_free > 0 && !a.free_pages) return invalid(who, "null free_pages");
    if (a.n_rows > 0 && (!a.positions || !a.slots)) return invalid(who, "null positions or slots");
    for (const void *p : {static_cast<const void *>(a.cached), static_cast<const void *>(a.added),
                          static_cast<const void *>(a.block_table), static_cast<const void *>(a.free_pages),
                          static_cast<const void *>(a.free_head), static_cast<const void *>(a.free_head_out),
                          static_cast<const void *>(a.row_offsets), static_cast<const void *>(a.kv_lens),
                          static_cast<const void *>(a.positions), static_cast<const void *>(a.status)})
        if (!aligned(p, 4)) return invalid(who, "pointers must be aligned to their values");
    if (!aligned(a.slots, 8)) return invalid(who, "pointers must be aligned to their values");
    if (int rc = device_gate(ctx, who)) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    if (take_fault("mi355x_kv_plan_pages")) {
        mi355x_kv_plan_args none = a;
        none.n_free = -1;  // no head lies in 0 .. -1: refused, whatever the step needs
        return launch_kv_plan(ctx, none);
    }
    return launch_kv_plan(ctx, a);
}

int mi355x_qk_norm_rope(mi355x_ctx *ctx, const mi355x_qk_norm_rope_args *args) {
    clear_error();
    static const char *who = "mi355x_qk_norm_rope";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_qk_norm_rope_args &a = *args;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (a.n_heads < 0 || a.n_kv_heads < 0 || a.n_heads > 65536 || a.n_kv_heads > 65536)
        return invalid(who, "n_heads and n_kv_heads must be 0 to 65536");
    if (a.head_dim < 2 || a.head_dim > 1024 || a.head_dim % 2 != 0)
        return invalid(who, "head_dim must be even and at most 1024 (got " + std::to_string(a.head_dim) + ")");
    if (a.rot_dim < 0 || a.rot_dim > a.head_dim || a.rot_dim % 2 != 0)
        return invalid(who, "rot_dim must be even and at most head_dim (got " + std::to_string(a.rot_dim) + ")");
    if (a.rope_mode != MI355X_ROPE_HALVES && a.rope_mode != MI355X_ROPE_PAIRS)
        return invalid(who, "unknown rope_mode " + std::to_string(a.rope_mode));
    const int ib = type_bytes(a.in_type), ob = type_bytes(a.out_type);
    if (!ib || !ob) return invalid(who, "in_type and out_type must be F32, F16 or BF16");
    if (!(a.eps >= 0.0f) || std::isinf(a.eps)) return invalid(who, "eps must be finite and not negative");
    const int64_t qw = static_cast<int64_t>(a.n_heads) * a.head_dim, kw = static_cast<int64_t>(a.n_kv_heads) * a.head_dim;
    if (a.pool) {
        if (int rc = check_pool(who, a.pool)) return rc;
        if (a.pool->type != a.out_type) return invalid(who, "out_type must be the pool's type");
        if (a.pool->head_dim != a.head_dim || a.pool->n_kv_heads != a.n_kv_heads)
            return invalid(who, "head_dim and n_kv_heads must be the pool's");
    }
    if (a.n_rows == 0 || a.n_heads + a.n_kv_heads == 0) return MI355X_OK;
    if (a.n_heads > 0) {
        if (!a.q || !a.q_out) return invalid(who, "null q or q_out");
        if (int rc = check_row_stride(who, "q_stride", a.n_rows, a.q_stride, qw)) return rc;
        if (int rc = check_row_stride(who, "q_out_stride", a.n_rows, a.q_out_stride, qw)) return rc;
        if (a.q_out == a.q && (a.in_type != a.out_type || a.q_stride != a.q_out_stride))
            return invalid(who, "q_out may be q only with q's type and stride");
    }
    if (a.n_kv_heads > 0) {
        if (!a.k) return invalid(who, "null k");
        if (int rc = check_row_stride(who, "k_stride", a.n_rows, a.k_stride, kw)) return rc;
        if (a.pool) {
            if (!a.v || !a.slots) return invalid(who, "null v or slots");
            if (int rc = check_row_stride(who, "v_stride", a.n_rows, a.v_stride, kw)) return rc;
        } else {
            if (!a.k_out) return invalid(who, "a pool or k_out is needed");
            if (int rc = check_row_stride(who, "k_out_stride", a.n_rows, a.k_out_stride, kw)) return rc;
            if (a.k_out == a.k && (a.in_type != a.out_type || a.k_stride != a.k_out_stride))
                return invalid(who, "k_out may be k only with k's type and stride");
        }
    }
    if (a.rot_dim > 0 && (!a.positions || !a.inv_freq)) return invalid(who, "null positions or inv_freq");
    for (const void *p : {a.q, a.k, a.pool ? a.v : nullptr})
        if (!aligned(p, static_cast<size_t>(ib))) return invalid(who, "pointers must be aligned to their values");
    for (const void *p : {static_cast<const void *>(a.q_out), a.pool ? nullptr : static_cast<const void *>(a.k_out)})
        if (!aligned(p, static_cast<size_t>(ob))) return invalid(who, "pointers must be aligned to their values");
    for (const void *p : {static_cast<const void *>(a.q_bias), static_cast<const void *>(a.k_bias),
                          static_cast<const void *>(a.v_bias), static_cast<const void *>(a.q_norm),
                          static_cast<const void *>(a.k_norm), static_cast<const void *>(a.positions),
                          static_cast<const void *>(a.inv_freq)})
        if (!aligned(p, 4)) return invalid(who, "pointers must be aligned to their values");
    if (a.pool && !aligned(a.slots, 8)) return invalid(who, "pointers must be aligned to their values");
    if (int rc = device_gate(ctx, who)) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_qk_norm_rope(ctx, a);
}

namespace {

// Head counts and sizes that mi355x_paged_attention computes.
int check_heads(const char *who, int n_heads, int n_kv_heads, int head_dim) {
    if (n_heads < 1 || n_heads > 65536 || n_kv_heads < 1 || n_heads % n_kv_heads != 0)
        return invalid(who, "n_heads must be a multiple of the pool's n_kv_heads, up to 65536 (got " +
                                std::to_string(n_heads) + " and " + std::to_string(n_kv_heads) + ")");
    if (head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 256)
        return set_error(MI355X_EUNSUPPORTED, std::string(who) + ": head_dim must be 64, 96, 128 or 256 (got " +
                                                  std::to_string(head_dim) + ")");
    return MI355X_OK;
}

}  // namespace

int mi355x_paged_attention_workspace(mi355x_ctx *ctx, int n_heads, int n_kv_heads, int head_dim, size_t *bytes) {
    clear_error();
    static const char *who = "mi355x_paged_attention_workspace";
    if (!ctx || !bytes) return invalid(who, "null pointer argument provided");
    if (int rc = check_heads(who, n_heads, n_kv_heads, head_dim)) return rc;
    if (int rc = device_gate(ctx, who)) return rc;
    *bytes = paged_attention_workspace_bytes(ctx, n_heads, n_kv_heads, head_dim);
    return MI355X_OK;
}

int mi355x_paged_attention(mi355x_ctx *ctx, const mi355x_paged_attention_args *args) {
    clear_error();
    static const char *who = "mi355x_paged_attention";
    if (!ctx || !args || !args->pool) return invalid(who, "null pointer argument provided");
    const mi355x_paged_attention_args &a = *args;
    if (int rc = check_pool(who, a.pool)) return rc;
    if (int rc = check_heads(who, a.n_heads, a.pool->n_kv_heads, a.pool->head_dim)) return rc;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (int rc = check_seqs(who, a.n_seqs)) return rc;
    if (a.max_added < 0) return invalid(who, "negative max_added");
    if (a.table_cols < 0 || a.table_stride < 0 || a.table_stride > INT32_MAX ||
        (a.n_seqs > 1 && a.table_stride < a.table_cols))
        return invalid(who, "table_stride must be at least table_cols and at most 2^31 - 1 (got " +
                                std::to_string(a.table_stride) + ")");
    if (static_cast<int64_t>(a.table_cols) * a.pool->page_tokens > (1 << 30))
        return invalid(who, "table_cols pages must hold at most 2^30 tokens");
    if (a.window < 0) return invalid(who, "negative window");
    if (!std::isfinite(a.scale)) return invalid(who, "scale must be finite");
    if (!(a.softcap >= 0.0f) || std::isinf(a.softcap)) return invalid(who, "softcap must be finite and not negative");
    if (a.out_type != a.pool->type && a.out_type != MI355X_TYPE_F32)
        return invalid(who, "out_type must be the pool's type or F32 (got " + std::to_string(a.out_type) + ")");
    if (a.n_rows * (a.n_heads / a.pool->n_kv_heads) > INT32_MAX)
        return invalid(who, "n_rows times the query heads of a KV head must be below 2^31");
    // a launch's threads are counted in 32 bits
    const int64_t blocks = (a.n_rows * (a.n_heads / a.pool->n_kv_heads) / 128 + a.n_seqs) * a.pool->n_kv_heads;
    if (blocks >= (1 << 23))
        return set_error(MI355X_EUNSUPPORTED, std::string(who) + ": " + std::to_string(blocks) +
                                                  " blocks of rows, 2^23 or more");
    const int64_t width = static_cast<int64_t>(a.n_heads) * a.pool->head_dim;
    if (int rc = check_row_stride(who, "q_stride", a.n_rows, a.q_stride, width)) return rc;
    if (int rc = check_row_stride(who, "out_stride", a.n_rows, a.out_stride, width)) return rc;
    if (a.q_stride % 8 != 0 || a.out_stride % 8 != 0) return invalid(who, "q_stride and out_stride must be multiples of 8");
    if (a.n_rows == 0 || a.n_seqs == 0) return MI355X_OK;
    if (!a.q || !a.out || !a.row_offsets || !a.kv_lens) return invalid(who, "null pointer argument provided");
    if (a.table_cols > 0 && !a.block_table) return invalid(who, "null block_table");
    if (!aligned(a.q, 16) || !aligned(a.out, 16)) return invalid(who, "q and out must be 16-byte aligned");
    for (const int32_t *p : {a.row_offsets, a.kv_lens, a.block_table})
        if (!aligned(p, 4)) return invalid(who, "pointers must be aligned to their values");
    if (int rc = device_gate(ctx, who)) return rc;
    const size_t need = paged_attention_workspace_bytes(ctx, a.n_heads, a.pool->n_kv_heads, a.pool->head_dim);
    if (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < need)
        return invalid(who, "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed (got " +
                                std::to_string(a.workspace ? a.workspace_bytes : 0) + ")");
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_paged_attention(ctx, a);
}

}  // extern "C"
