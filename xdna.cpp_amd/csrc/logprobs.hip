// Log probabilities of given tokens, entropy and top tokens of rows of logits.
//
// With m the row's largest logit and d_i = scale (m - x_i) >= 0: S = sum exp(-d_i),
// log p_i = -d_i - log S, entropy = log S + sum exp(-d_i) d_i / S, every term of
// either sum of one sign.
#include "internal.h"
#include "row_values.h"

#include <algorithm>
#include <cfloat>

namespace mi355x {
namespace {

struct LogitArgs {
    int64_t n_rows, stride;
    const void *logits;
    int n_vocab, type, n_tokens, n_top;
    float scale;
    const int32_t *tokens;
    float *token_logprobs, *entropy, *top_logprobs;
    int32_t *top_tokens;
};

constexpr int kThreads = 256;

__device__ __forceinline__ float logit(const LogitArgs &a, int64_t row, int i) {
    const int64_t at = row * a.stride + i;
    if (a.type == MI355X_TYPE_F32) return static_cast<const float *>(a.logits)[at];
    if (a.type == MI355X_TYPE_F16) return static_cast<float>(static_cast<const _Float16 *>(a.logits)[at]);
    return static_cast<float>(static_cast<const __bf16 *>(a.logits)[at]);
}

// The larger logit, of equal ones the lower token.
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogitArgs a) {
    __shared__ float lds_f[kThreads], lds_g[kThreads];
    __shared__ int lds_i[kThreads];
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
        // the first top token is the row's largest logit
        float last = INFINITY, top = -INFINITY, log_total = 0.0f;
        int last_i = -1;
        bool bad = false;
        for (int r = 0; r < max(a.n_top, 1); ++r) {
            float x = -INFINITY;
            int at = INT_MAX;
            for (int i = tid; i < a.n_vocab; i += kThreads) {
                const float v = logit(a, row, i);
                if (r == 0) bad |= !(v < INFINITY);
                if (v > -INFINITY && before(v, i, x, at) && before(last, last_i, v, i)) {
                    x = v;
                    at = i;
                }
            }
            lds_f[tid] = x;
            lds_i[tid] = at;
            if (r == 0) bad = __syncthreads_or(bad);
            else __syncthreads();
            for (int t = 0; t < kThreads; ++t)
                if (before(lds_f[t], lds_i[t], x, at)) {
                    x = lds_f[t];
                    at = lds_i[t];
                }
            __syncthreads();
            if (r == 0) {
                top = x;
                float s = 0.0f, e = 0.0f;
                for (int i = tid; i < a.n_vocab; i += kThreads) {
                    const float d = a.scale * (top - logit(a, row, i)), p = expf(-d);
                    s += p;
                    if (p > 0.0f) e += p * d;
                }
                lds_f[tid] = s;
                lds_g[tid] = e;
                __syncthreads();
                s = e = 0.0f;
                for (int t = 0; t < kThreads; ++t) {
                    s += lds_f[t];
                    e += lds_g[t];
                }
                __syncthreads();
                const bool none = top == -INFINITY;
                log_total = bad ? NAN : none ? 0.0f : logf(s);
                if (a.entropy && tid == 0) a.entropy[row] = bad ? NAN : none ? 0.0f : log_total + e / s;
                for (int t = tid; t < a.n_tokens; t += kThreads) {
                    const int token = a.tokens[row * a.n_tokens + t];
                    const bool in = token >= 0 && token < a.n_vocab;
                    const float v = in ? logit(a, row, token) : 0.0f;
                    a.token_logprobs[row * a.n_tokens + t] =
                        bad || !in ? NAN : v == -INFINITY ? v : a.scale * (v - top) - log_total;
                }
            }
            if (tid == 0 && r < a.n_top) {
                const bool none = at == INT_MAX;
                a.top_tokens[row * a.n_top + r] = bad || none ? -1 : at;
                a.top_logprobs[row * a.n_top + r] = bad ? NAN : none ? -INFINITY : a.scale * (x - top) - log_total;
            }
            last = x;
            last_i = at;
        }
    }
}

}  // namespace

size_t logprobs_workspace_bytes(const mi355x_ctx *ctx) { return static_cast<size_t>(ctx->num_cus) * 4096 + 65536; }

int launch_logprobs(mi355x_ctx *ctx, const mi355x_logprobs_args &u) {
    LogitArgs a{};
    a.n_rows = u.n_rows;
    a.stride = u.stride;
    a.logits = u.logits;
    a.n_vocab = u.n_vocab;
    a.type = u.type;
    a.n_tokens = u.n_tokens;
    a.n_top = u.n_top;
    a.scale = u.scale;
    a.tokens = u.tokens;
    a.token_logprobs = u.token_logprobs;
    a.entropy = u.entropy;
    a.top_logprobs = u.top_logprobs;
    a.top_tokens = u.top_tokens;
    logprobs_kernel<<<static_cast<unsigned>(std::min<int64_t>(u.n_rows, 1 << 20)), kThreads, 0, ctx->stream>>>(a);
    MI355X_HIP(hipGetLastError());
    return MI355X_OK;
}

}  // namespace mi355x
