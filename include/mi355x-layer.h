/*
 * mi355x-layer.h -- a layer's rows and products in 8-bit integers, and what a
 * model's logits are read for.
 *
 * They stand beside the GEMVs of mi355x-gemv.h and the attention of
 * mi355x-attention.h, and are called in the same manner: plain pointers and
 * sizes, a context that carries the device and the stream, the MI355X_* status
 * codes, mi355x_last_error().  Every call checks what the host can see, enqueues
 * on the context's stream and returns; pointers in the argument blocks are device
 * addresses, aligned to their values; the blocks themselves are read during the
 * call.  Nothing is allocated, so every call may be recorded into a HIP graph.
 * Strides are in values.  Nothing behind a row's values is written, and outputs
 * may not overlap inputs or each other but where it says so.
 *
 * No counterpart in the reference, which runs MUL_MAT of 4-bit weights and leaves
 * norms, gates and logits to ggml-cpu (src/ggml-xdna.cpp:95-147, 783-823).
 *
 * A layer with 8-bit weights: mi355x_norm_q8, the q|k|v product, the operators
 * of mi355x-attention.h, mi355x_norm_q8 without a norm on their output, the o
 * product, mi355x_norm_q8 with the residual, the gate|up product,
 * mi355x_swiglu_q8, the down product.  Behind the last layer mi355x_norm_q8, the
 * vocabulary product, mi355x_logprobs.
 */
#ifndef MI355X_LAYER_H
#define MI355X_LAYER_H

#include "mi355x-attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rows in 8 bits -----------------------------------------------------------
 * A row of values t_0 .. t_n-1 is held as codes and a scale, t_i ~ scale * code_i:
 *   code_i = t_i * 127 / max_j |t_j|, rounded to nearest, ties to even, -127 .. 127
 *   scale  = max_j |t_j| / 127, rounded to f32 (infinite past f32's range)
 * The t_i, the product and the quotient are 64-bit numbers, so that a code is not
 * off where its quotient lies next to a border.  A row of zeros has codes and scale
 * 0.  A row with a t_i that is infinite or NaN has codes 0 and the scale NaN, so
 * that its products are NaN. */

/* The residual's addition, the root-mean-square norm, and the row in 8 bits:
 *   h_i = x_i + residual_i, in f32, rounded to residual_type (without a residual
 *         h_i = x_i as it is); stored in residual_out where one is given
 *   t_i = h_i * norm_i / sqrt(mean_j(h_j^2) + eps)
 * The mean is summed in 64 bits.  The root, which a whole row has in common, meets the
 * scale alone: codes are those of the products h_i * norm_i (64-bit numbers, exact), so
 * that a tie of theirs is a tie whatever the root rounds to.  Without norm t_i = h_i:
 * rows are only put in 8 bits, and eps is not used (it is checked all the same).  So a
 * weight of 16 or 32 bits, its channels as rows, becomes the w and w_scales of
 * mi355x_matmul_q8.  residual_out may be residual or x (same type and stride as
 * that). */
#define MI355X_ROW_Q8_MAX 65536
typedef struct mi355x_norm_q8_args {
    int64_t n_rows;       /* at most 2^31 - 1 */
    int n;                /* values of a row, 1 .. MI355X_ROW_Q8_MAX */
    int type;             /* x: MI355X_TYPE_F32, _F16 or _BF16 */
    const void *x;
    int64_t x_stride;
    int residual_type;    /* residual and residual_out (not used without a residual) */
    float eps;            /* finite, not negative */
    const void *residual; /* or NULL */
    int64_t residual_stride;
    void *residual_out;   /* or NULL; NULL without a residual */
    int64_t residual_out_stride;
    const float *norm;    /* n, or NULL */
    int8_t *q;
    int64_t q_stride;
    float *scales;        /* n_rows */
} mi355x_norm_q8_args;
MI355X_API int mi355x_norm_q8(mi355x_ctx *ctx, const mi355x_norm_q8_args *args);

/* A gated row in 8 bits: t_i = gate_i / (1 + exp(-gate_i)) * up_i, formed in 64
 * bits (an infinite gate is a t that is not finite).  gate and up may be halves
 * of one row. */
typedef struct mi355x_swiglu_q8_args {
    int64_t n_rows; /* at most 2^31 - 1 */
    int n;          /* 1 .. MI355X_ROW_Q8_MAX */
    int type;       /* gate, up: MI355X_TYPE_F32, _F16 or _BF16 */
    const void *gate;
    int64_t gate_stride;
    const void *up;
    int64_t up_stride;
    int8_t *q;
    int64_t q_stride;
    float *scales;  /* n_rows */
} mi355x_swiglu_q8_args;
MI355X_API int mi355x_swiglu_q8(mi355x_ctx *ctx, const mi355x_swiglu_q8_args *args);

/* ---- products of 8-bit integers -------------------------------------------------
 *   out[m][o] = (sum_c x[m][c] * w[o][c]) * w_scales[o] * x_scales[m] + bias[o]
 * for m < n_rows, o < n_out, c < k.  The sum is exact in 32-bit integers (codes
 * may be -128); it is rounded to f32, multiplied and added to in f32 in this
 * order, and rounded once to out_type.  x, w: 16-byte aligned, rows of a multiple
 * of 16 codes, strides multiples of 16.  The result does not depend on how the
 * work is split.  MI355X_EUNSUPPORTED: 2^34 outputs or more, and more than 64 *
 * 65535 rows where a stride passes 2^23.
 *
 * workspace: mi355x_matmul_q8_workspace bytes, 16-byte aligned.  Zero it once,
 * before its first call (mi355x_fill): it begins with counters that every call
 * finds and leaves at 0.  Calls that may run at the same time (two contexts, a
 * graph replayed beside other calls, two graphs) need one each; calls in order on
 * one stream share one, but not with other operators. */
#define MI355X_MATMUL_Q8_MAX_K 131056
typedef struct mi355x_matmul_q8_args {
    int64_t n_rows; /* at most 2^24 */
    int64_t n_out;  /* at most 2^24 */
    int64_t k;      /* a multiple of 16, up to MI355X_MATMUL_Q8_MAX_K */
    const int8_t *x;
    int64_t x_stride;
    const float *x_scales; /* n_rows */
    const int8_t *w;
    int64_t w_stride;
    const float *w_scales; /* n_out */
    const float *bias;     /* n_out, or NULL */
    void *out;
    int out_type;          /* MI355X_TYPE_F32, _F16 or _BF16 */
    int64_t out_stride;
    void *workspace;
    size_t workspace_bytes;
} mi355x_matmul_q8_args;
MI355X_API int mi355x_matmul_q8(mi355x_ctx *ctx, const mi355x_matmul_q8_args *args);
/* Bytes of workspace that any call needs on the context's device. */
MI355X_API int mi355x_matmul_q8_workspace(mi355x_ctx *ctx, size_t *bytes);

/* ---- log probabilities of logits -----------------------------------------------
 * For each row x_0 .. x_V-1 of logits, with p_i = exp(scale * x_i) / sum_j exp(scale * x_j):
 *   token_logprobs[row][t] = log p of token tokens[row][t]  (NaN for one outside 0 .. V - 1)
 *   entropy[row] = - sum_i p_i log p_i                       (natural logarithms)
 *   top_tokens[row][r] = the token of the r-th largest logit, equal ones in ascending
 *     order of the token; top_logprobs[row][r] its log p
 * in f32 with the row's largest logit taken out first, in one pass over the row.
 * A logit of -inf has p = 0 and log p = -inf, adds nothing to the entropy and is no
 * top token: where fewer than n_top others are left, -1 and -inf stand in their
 * place.  A row of -inf alone has -inf for every token, and the entropy 0.  A row
 * with NaN or +inf has NaN for everything, and -1 for every top token.  Tokens that are
 * not allowed are best given -inf: where more than 1024 logits above -inf are as large as
 * the last top token's less 2^-7 of its size (a finite lowest value on all but a few, or a
 * common offset of a hundred times their spread), the row is read n_top times.
 *
 * workspace: mi355x_logprobs_workspace bytes, under the same rules as that of
 * mi355x_matmul_q8. */
#define MI355X_LOGPROBS_MAX_TOP 64
typedef struct mi355x_logprobs_args {
    int64_t n_rows;  /* at most 2^31 - 1 */
    int n_vocab;     /* V, 1 .. 2^30 */
    int type;        /* logits: MI355X_TYPE_F32, _F16 or _BF16 */
    const void *logits;
    int64_t stride;
    float scale;     /* 1 / temperature: 2^-100 .. 2^100 */
    int n_tokens;    /* of each row, 0 .. 65536 */
    const int32_t *tokens;  /* n_rows * n_tokens */
    float *token_logprobs;  /* n_rows * n_tokens */
    float *entropy;         /* n_rows, or NULL */
    int n_top;              /* 0 .. MI355X_LOGPROBS_MAX_TOP */
    int32_t *top_tokens;    /* n_rows * n_top */
    float *top_logprobs;    /* n_rows * n_top */
    void *workspace;
    size_t workspace_bytes;
} mi355x_logprobs_args;
MI355X_API int mi355x_logprobs(mi355x_ctx *ctx, const mi355x_logprobs_args *args);
/* Bytes of workspace that any call needs on the context's device. */
MI355X_API int mi355x_logprobs_workspace(mi355x_ctx *ctx, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif
