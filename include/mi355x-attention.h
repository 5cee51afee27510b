/*
 * mi355x-attention.h -- the operators between a layer's q|k|v projection and
 * its output projection, over a paged KV cache.
 *
 * They stand beside the GEMVs of mi355x-gemv.h and share their manner: plain
 * pointers and sizes, a context that carries the device and the stream, the
 * MI355X_* status codes, mi355x_last_error().  Every call checks what the host
 * can see, enqueues on the context's stream and returns; every pointer in an
 * argument block is a device address unless it is marked "host".  The blocks
 * themselves are read during the call.  Nothing is allocated, so every call
 * may be recorded into a HIP graph; lengths, tables and positions are device
 * memory, so that a graph's replays take new ones.
 *
 * No counterpart in the reference, which runs MUL_MAT alone and leaves
 * attention to ggml-cpu (src/ggml-xdna.cpp:95-147, 783-823).
 *
 * A step of a serving loop is one mi355x_kv_plan (which pages and slots the
 * new tokens take), then in each layer the q|k|v GEMV, mi355x_qk_norm_rope
 * (bias, norms, rotation; keys and values into their slots),
 * mi355x_paged_attention, and the output GEMV.  The new tokens of all requests
 * lie one behind the other as rows; request s has rows
 * row_offsets[s] .. row_offsets[s + 1] - 1 and they are the last ones of its
 * kv_lens[s] tokens.
 */
#ifndef MI355X_ATTENTION_H
#define MI355X_ATTENTION_H

#include "mi355x-gemv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ggml's type ids of the 16-bit floats (MI355X_TYPE_F32 is in mi355x-gemv.h) */
#define MI355X_TYPE_F16 1
#define MI355X_TYPE_BF16 30

/* One layer's pages of keys and values.  Token t of a request whose table has
 * page p at column t / page_tokens lies at
 *   k + p * page_stride + (t % page_tokens) * token_stride + h * head_stride
 * (strides in values) for head h, head_dim values side by side; so do the
 * values, from v.  [page][token][head] and [page][head][token] are both
 * strides of this kind.  k, v: 16-byte aligned; strides: multiples of 8, at most
 * 2^31. */
typedef struct mi355x_kv_pool {
    int type;        /* MI355X_TYPE_F16 or MI355X_TYPE_BF16 */
    int n_kv_heads;
    int head_dim;
    int page_tokens; /* a power of two, at most 65536 */
    int64_t n_pages; /* at most 2^31 - 1 */
    void *k;
    void *v;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
} mi355x_kv_pool;

/* ---- block tables and slots -------------------------------------------------
 * From each request's cached tokens and the ones it adds:
 *   row_offsets[s] = added[0] + .. + added[s - 1]   (n_seqs + 1 entries)
 *   kv_lens[s]     = cached[s] + added[s]
 *   block_table[s][c] for the columns c in [ceil(cached / page_tokens),
 *     ceil(kv_len / page_tokens)) = the next unused entries of free_pages, from
 *     entry *free_head on, requests in order
 *   *free_head_out = *free_head + the entries taken
 *   row r of request s, i = r - row_offsets[s]: positions[r] = cached[s] + i,
 *     slots[r] = page * page_tokens + positions[r] % page_tokens with the page
 *     that the table has for it
 *   rows behind the last request's, up to n_rows: position 0 and slot -1
 * All or nothing: where a length is negative or a sum of two passes 2^31 - 1,
 * the rows, the table's columns or the free pages do not suffice, *status is
 * the sum of the MI355X_KV_* bits that say so, no page is taken, row_offsets
 * are all 0, kv_lens are the cached lengths (0 for a negative one) and every
 * slot is -1, so that the operators behind it do nothing; else *status is 0.
 * free_head_out may be free_head, and kv_lens may be cached; nothing else may
 * overlap.  status may be NULL. */
#define MI355X_KV_BAD_LENGTH 1  /* a negative length, or a sum past 2^31 - 1 */
#define MI355X_KV_ROWS 2        /* more new tokens than n_rows */
#define MI355X_KV_TABLE 4       /* a request needs more than table_cols pages */
#define MI355X_KV_PAGES 8       /* fewer free pages than needed (or *free_head not in 0 .. n_free) */
typedef struct mi355x_kv_plan_args {
    int n_seqs;            /* requests, at most 65536 */
    int page_tokens;       /* a power of two, at most 65536 */
    int table_cols;
    int n_free;            /* entries of free_pages */
    int64_t table_stride;  /* entries from one request's table row to the next */
    int64_t n_rows;        /* entries of positions and slots, at most 2^31 - 1 */
    const int32_t *cached; /* n_seqs */
    const int32_t *added;  /* n_seqs */
    int32_t *block_table;
    const int32_t *free_pages;
    const int32_t *free_head;
    int32_t *free_head_out;
    int32_t *row_offsets;  /* n_seqs + 1 */
    int32_t *kv_lens;      /* n_seqs */
    int32_t *positions;    /* n_rows */
    int64_t *slots;        /* n_rows */
    int32_t *status;
} mi355x_kv_plan_args;
MI355X_API int mi355x_kv_plan(mi355x_ctx *ctx, const mi355x_kv_plan_args *args);

/* ---- norms of queries and keys, rotation, store --------------------------------
 * For every row and every head of q, k and v (head h at h * head_dim):
 *   x = in + bias                                  (q, k, v; where a bias is given)
 *   x = x / sqrt(mean(x^2) + eps) * norm           (q, k; where a norm is given)
 *   with a_i, b_i the pairs of the first rot_dim values -- MI355X_ROPE_HALVES:
 *   x[i], x[i + rot_dim / 2]; MI355X_ROPE_PAIRS: x[2 i], x[2 i + 1] -- and
 *   angle = positions[row] * inv_freq[i]:          (q, k)
 *   a_i, b_i = a_i cos - b_i sin, b_i cos + a_i sin
 * in f32, the angle in 64 bits, each result rounded once to out_type.  Queries
 * go to q_out; keys and values to slot slots[row] of the pool (out_type is the
 * pool's type then), and a row whose slot is not in the pool (-1, say) stores
 * neither.  Without a pool keys go to k_out, and v, v_bias, v_stride and slots
 * are not used.  No two rows may have the same slot.  q_out and k_out may be q
 * and k (same type and stride); nothing else may overlap. */
#define MI355X_ROPE_HALVES 0
#define MI355X_ROPE_PAIRS 1
typedef struct mi355x_qk_norm_rope_args {
    int64_t n_rows;          /* at most 2^31 - 1 */
    int n_heads;
    int n_kv_heads;
    int head_dim;            /* even, at most 1024 (with a pool: a multiple of 8) */
    int rot_dim;             /* even, 0 .. head_dim */
    int rope_mode;
    int in_type;             /* MI355X_TYPE_F32, _F16 or _BF16: q, k, v */
    int out_type;            /* MI355X_TYPE_F16 or _BF16 (without a pool also _F32) */
    float eps;
    const void *q, *k, *v;   /* first row; the next one *_stride values on */
    int64_t q_stride, k_stride, v_stride;
    const float *q_bias, *k_bias, *v_bias; /* heads * head_dim each, or NULL */
    const float *q_norm, *k_norm;          /* head_dim each, or NULL */
    const int32_t *positions;              /* n_rows (NULL allowed if rot_dim is 0) */
    const float *inv_freq;                 /* rot_dim / 2 (NULL allowed if rot_dim is 0) */
    void *q_out;
    int64_t q_out_stride;
    const mi355x_kv_pool *pool;            /* host; or NULL */
    const int64_t *slots;                  /* n_rows */
    void *k_out;
    int64_t k_out_stride;
} mi355x_qk_norm_rope_args;
MI355X_API int mi355x_qk_norm_rope(mi355x_ctx *ctx, const mi355x_qk_norm_rope_args *args);

/* ---- attention over the pages ---------------------------------------------------
 * Row i of request s, n = row_offsets[s + 1] - row_offsets[s], has position
 * p = kv_lens[s] - n + i; its head h attends with the KV head
 * h / (n_heads / n_kv_heads) to the request's tokens
 *   j <= p (causal != 0; else every j < kv_lens[s]),  and j > p - window (window > 0):
 *   score_j = scale * q . k_j;  softcap > 0: softcap * tanh(score_j / softcap)
 *   out = sum_j exp(score_j - max) v_j / sum_j exp(score_j - max)
 * Scores, weights and sums are f32 (capped scores to 2^-23 of the cap), products of
 * 16-bit values on the matrix cores.  The weights meet v as 16-bit values of the pool's type (half a step,
 * 2^-8 or 2^-11 of a weight: as much as the rounding of a 16-bit output), or
 * as two such planes (no more than 2^-16 of a weight then) where the request takes
 * the form for few rows: at most 16 of them times query heads of a KV head, by
 * max_added or, in a call of several requests, its own.  With an f32 output they go in
 * to 2^-22, in as many planes as that takes.  F16 has steps of 2^-24 besides: weights
 * are off by up to 2^-24 of the largest one among the 32 or 64 tokens that they are
 * taken with, and by more below 2^-40 of the row's largest.
 * A row that sees nothing gives zeros.  Tokens that a row does not see do not
 * reach its output, whatever their bits are (NaN and infinities too), and
 * columns of the table that no row of the request sees are not read.  An infinite
 * value of v that a row sees makes that value of its output infinite or NaN (with more
 * than one plane NaN also where all such have one sign), and no other.  Tokens on
 * a page outside the pool (a table entry not in 0 .. n_pages - 1), behind the
 * table's last column or of a negative length count as not seen.  Rows of out
 * behind row_offsets[n_seqs], and rows that offsets past n_rows name, are not
 * written.  row_offsets ascend from 0.
 * head_dim 64, 96, 128 or 256 (others: MI355X_EUNSUPPORTED, and so are 2^23
 * blocks of rows: (n_rows * group / 128 + n_seqs) * n_kv_heads); q, out: 16-byte
 * aligned rows (q_stride a multiple of 8, out_stride of 8), head h at
 * h * head_dim; out may not overlap an input.  max_added is the host's bound on
 * a request's new tokens (0: unknown); it picks the form, and with it the number of
 * planes, and never which rows are computed.
 *
 * workspace: mi355x_paged_attention_workspace bytes for parts of long rows,
 * 16-byte aligned.  Zero it once, before its first call (mi355x_fill): it
 * begins with counters that every call finds and leaves at 0.  Calls that may
 * run at the same time (two contexts, a graph replayed beside other calls, two
 * graphs) need one each; calls in order on one stream share one. */
typedef struct mi355x_paged_attention_args {
    int64_t n_rows;           /* rows of q and out; times n_heads / n_kv_heads at most 2^31 - 1 */
    int n_seqs;               /* at most 65536 */
    int n_heads;              /* a multiple of the pool's n_kv_heads */
    int max_added;
    const void *q;            /* the pool's type */
    int64_t q_stride;         /* values between rows */
    const mi355x_kv_pool *pool; /* host */
    const int32_t *row_offsets; /* n_seqs + 1 */
    const int32_t *kv_lens;     /* n_seqs */
    const int32_t *block_table;
    int table_cols;           /* times page_tokens at most 2^30 */
    int64_t table_stride;
    float scale;
    float softcap;            /* 0: none */
    int window;               /* 0: none */
    int causal;
    void *out;
    int out_type;             /* the pool's type or MI355X_TYPE_F32 */
    int64_t out_stride;
    void *workspace;
    size_t workspace_bytes;
} mi355x_paged_attention_args;
MI355X_API int mi355x_paged_attention(mi355x_ctx *ctx, const mi355x_paged_attention_args *args);
/* Bytes of workspace that any call with these heads needs on the context's device. */
MI355X_API int mi355x_paged_attention_workspace(mi355x_ctx *ctx, int n_heads, int n_kv_heads, int head_dim,
                                                size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif
