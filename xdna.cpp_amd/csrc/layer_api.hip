// Entry points of mi355x-layer.h: what the host can check of a call's
// arguments, the device gate, and the launch.
#include "internal.h"

#include <climits>
#include <cmath>
#include <string>

namespace mi355x {
namespace {

int invalid(const char *who, const std::string &what) {
    return set_error(MI355X_EINVAL, std::string(who) + ": " + what);
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int type_bytes(int type) {
    return type == MI355X_TYPE_F32 ? 4 : type == MI355X_TYPE_F16 || type == MI355X_TYPE_BF16 ? 2 : 0;
}

int check_rows(const char *who, int64_t n) {
    if (n < 0 || n > INT32_MAX) return invalid(who, "n_rows must be 0 to 2^31 - 1 (got " + std::to_string(n) + ")");
    return MI355X_OK;
}

int check_type(const char *who, const char *name, int type) {
    if (!type_bytes(type))
        return invalid(who, std::string(name) + " must be F32, F16 or BF16 (got " + std::to_string(type) + ")");
    return MI355X_OK;
}

// Rows of `width` values, `bytes` each, `stride` values apart.
int check_rows_at(const char *who, const char *name, const void *p, int bytes, int64_t n, int64_t stride,
                  int64_t width) {
    if (!p) return invalid(who, std::string("null ") + name);
    if (!aligned(p, static_cast<size_t>(bytes)))
        return invalid(who, std::string(name) + " must be " + std::to_string(bytes) + "-byte aligned");
    if (stride < 0 || stride > (int64_t(1) << 40) || (n > 1 && stride < width))
        return invalid(who, std::string(name) + "'s stride must be at least a row's " + std::to_string(width) +
                                " values and at most 2^40 (got " + std::to_string(stride) + ")");
    return MI355X_OK;
}

int check_vector(const char *who, const char *name, const void *p) {
    if (!p) return invalid(who, std::string("null ") + name);
    if (!aligned(p, 4)) return invalid(who, std::string(name) + " must be 4-byte aligned");
    return MI355X_OK;
}

int check_row_values(const char *who, int n) {
    if (n < 1 || n > MI355X_ROW_Q8_MAX)
        return invalid(who, "n must be 1 to " + std::to_string(MI355X_ROW_Q8_MAX) + " (got " + std::to_string(n) + ")");
    return MI355X_OK;
}

int check_workspace(const char *who, const void *p, size_t bytes, size_t need) {
    if (!p || !aligned(p, 16) || bytes < need)
        return invalid(who, "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed (got " +
                                std::to_string(p ? bytes : 0) + ")");
    return MI355X_OK;
}

}  // namespace
}  // namespace mi355x

using namespace mi355x;

extern "C" {

int mi355x_norm_q8(mi355x_ctx *ctx, const mi355x_norm_q8_args *args) {
    clear_error();
    static const char *who = "mi355x_norm_q8";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_norm_q8_args &a = *args;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (int rc = check_row_values(who, a.n)) return rc;
    if (int rc = check_type(who, "type", a.type)) return rc;
    if (a.residual)
        if (int rc = check_type(who, "residual_type", a.residual_type)) return rc;
    if (!a.residual && a.residual_out) return invalid(who, "residual_out without a residual");
    if (!(a.eps >= 0.0f) || std::isinf(a.eps)) return invalid(who, "eps must be finite and not negative");
    if (a.n_rows == 0) return MI355X_OK;
    if (int rc = check_rows_at(who, "x", a.x, type_bytes(a.type), a.n_rows, a.x_stride, a.n)) return rc;
    if (a.residual) {
        const int rb = type_bytes(a.residual_type);
        if (int rc = check_rows_at(who, "residual", a.residual, rb, a.n_rows, a.residual_stride, a.n)) return rc;
        if (a.residual_out) {
            if (int rc = check_rows_at(who, "residual_out", a.residual_out, rb, a.n_rows, a.residual_out_stride, a.n))
                return rc;
            if (a.residual_out == a.residual && a.n_rows > 1 && a.residual_out_stride != a.residual_stride)
                return invalid(who, "residual_out may be residual only with its stride");
            if (a.residual_out == a.x &&
                (a.type != a.residual_type || (a.n_rows > 1 && a.residual_out_stride != a.x_stride)))
                return invalid(who, "residual_out may be x only with x's type and stride");
        }
    }
    if (a.norm)
        if (int rc = check_vector(who, "norm", a.norm)) return rc;
    if (int rc = check_rows_at(who, "q", a.q, 1, a.n_rows, a.q_stride, a.n)) return rc;
    if (int rc = check_vector(who, "scales", a.scales)) return rc;
    if (int rc = device_gate(ctx, who)) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_norm_q8(ctx, a);
}

int mi355x_swiglu_q8(mi355x_ctx *ctx, const mi355x_swiglu_q8_args *args) {
    clear_error();
    static const char *who = "mi355x_swiglu_q8";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_swiglu_q8_args &a = *args;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (int rc = check_row_values(who, a.n)) return rc;
    if (int rc = check_type(who, "type", a.type)) return rc;
    if (a.n_rows == 0) return MI355X_OK;
    if (int rc = check_rows_at(who, "gate", a.gate, type_bytes(a.type), a.n_rows, a.gate_stride, a.n)) return rc;
    if (int rc = check_rows_at(who, "up", a.up, type_bytes(a.type), a.n_rows, a.up_stride, a.n)) return rc;
    if (int rc = check_rows_at(who, "q", a.q, 1, a.n_rows, a.q_stride, a.n)) return rc;
    if (int rc = check_vector(who, "scales", a.scales)) return rc;
    if (int rc = device_gate(ctx, who)) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_swiglu_q8(ctx, a);
}

int mi355x_matmul_q8_workspace(mi355x_ctx *ctx, size_t *bytes) {
    clear_error();
    static const char *who = "mi355x_matmul_q8_workspace";
    if (!ctx || !bytes) return invalid(who, "null pointer argument provided");
    if (int rc = device_gate(ctx, who)) return rc;
    *bytes = matmul_q8_workspace_bytes(ctx);
    return MI355X_OK;
}

int mi355x_matmul_q8(mi355x_ctx *ctx, const mi355x_matmul_q8_args *args) {
    clear_error();
    static const char *who = "mi355x_matmul_q8";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_matmul_q8_args &a = *args;
    constexpr int64_t kMost = int64_t(1) << 24;
    if (a.n_rows < 0 || a.n_rows > kMost || a.n_out < 0 || a.n_out > kMost)
        return invalid(who, "n_rows and n_out must be 0 to 2^24 (got " + std::to_string(a.n_rows) + " and " +
                                std::to_string(a.n_out) + ")");
    if (a.k < 16 || a.k > MI355X_MATMUL_Q8_MAX_K || a.k % 16 != 0)
        return invalid(who, "k must be a multiple of 16 up to " + std::to_string(MI355X_MATMUL_Q8_MAX_K) + " (got " +
                                std::to_string(a.k) + ")");
    if (int rc = check_type(who, "out_type", a.out_type)) return rc;
    if (a.n_rows == 0 || a.n_out == 0) return MI355X_OK;
    if (int rc = check_rows_at(who, "x", a.x, 16, a.n_rows, a.x_stride, a.k)) return rc;
    if (int rc = check_rows_at(who, "w", a.w, 16, a.n_out, a.w_stride, a.k)) return rc;
    if (a.x_stride % 16 != 0 || a.w_stride % 16 != 0)
        return invalid(who, "x_stride and w_stride must be multiples of 16");
    if (a.n_rows * a.n_out >= int64_t(1) << 34)
        return set_error(MI355X_EUNSUPPORTED, std::string(who) + ": 2^34 outputs or more");
    // (a grid's second side has 16 bits)
    if (a.n_rows > 64 * 65535 && (a.x_stride > (1 << 23) || a.w_stride > (1 << 23)))
        return set_error(MI355X_EUNSUPPORTED, std::string(who) + ": more than 64 * 65535 rows with a stride past 2^23");
    if (int rc = check_vector(who, "x_scales", a.x_scales)) return rc;
    if (int rc = check_vector(who, "w_scales", a.w_scales)) return rc;
    if (a.bias)
        if (int rc = check_vector(who, "bias", a.bias)) return rc;
    if (int rc = check_rows_at(who, "out", a.out, type_bytes(a.out_type), a.n_rows, a.out_stride, a.n_out)) return rc;
    if (int rc = device_gate(ctx, who)) return rc;
    if (int rc = check_workspace(who, a.workspace, a.workspace_bytes, matmul_q8_workspace_bytes(ctx))) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_matmul_q8(ctx, a);
}

int mi355x_logprobs_workspace(mi355x_ctx *ctx, size_t *bytes) {
    clear_error();
    static const char *who = "mi355x_logprobs_workspace";
    if (!ctx || !bytes) return invalid(who, "null pointer argument provided");
    if (int rc = device_gate(ctx, who)) return rc;
    *bytes = logprobs_workspace_bytes(ctx);
    return MI355X_OK;
}

int mi355x_logprobs(mi355x_ctx *ctx, const mi355x_logprobs_args *args) {
    clear_error();
    static const char *who = "mi355x_logprobs";
    if (!ctx || !args) return invalid(who, "null pointer argument provided");
    const mi355x_logprobs_args &a = *args;
    if (int rc = check_rows(who, a.n_rows)) return rc;
    if (a.n_vocab < 1 || a.n_vocab > (1 << 30))
        return invalid(who, "n_vocab must be 1 to 2^30 (got " + std::to_string(a.n_vocab) + ")");
    if (int rc = check_type(who, "type", a.type)) return rc;
    // (a multiple of it by log2 e, and quotients by it, stay in f32's range)
    if (!(a.scale >= 0x1p-100f && a.scale <= 0x1p100f)) return invalid(who, "scale must be 2^-100 to 2^100");
    if (a.n_tokens < 0 || a.n_tokens > 65536) return invalid(who, "n_tokens must be 0 to 65536");
    if (a.n_top < 0 || a.n_top > MI355X_LOGPROBS_MAX_TOP)
        return invalid(who, "n_top must be 0 to " + std::to_string(MI355X_LOGPROBS_MAX_TOP) + " (got " +
                                std::to_string(a.n_top) + ")");
    if (a.n_rows == 0 || (a.n_tokens == 0 && a.n_top == 0 && !a.entropy)) return MI355X_OK;
    if (int rc = check_rows_at(who, "logits", a.logits, type_bytes(a.type), a.n_rows, a.stride, a.n_vocab)) return rc;
    if (a.n_tokens > 0) {
        if (int rc = check_vector(who, "tokens", a.tokens)) return rc;
        if (int rc = check_vector(who, "token_logprobs", a.token_logprobs)) return rc;
    }
    if (a.entropy)
        if (int rc = check_vector(who, "entropy", a.entropy)) return rc;
    if (a.n_top > 0) {
        if (int rc = check_vector(who, "top_tokens", a.top_tokens)) return rc;
        if (int rc = check_vector(who, "top_logprobs", a.top_logprobs)) return rc;
    }
    if (int rc = device_gate(ctx, who)) return rc;
    if (int rc = check_workspace(who, a.workspace, a.workspace_bytes, logprobs_workspace_bytes(ctx))) return rc;
    DeviceGuard dg(ctx->device);
    if (int rc = ov_join(ctx)) return rc;
    return launch_logprobs(ctx, a);
}

}  // extern "C"
