/*
 * lcml_decode_step.h — C ABI of what a decoder's step needs beside the norm, the
 * cache and the attention of lcml_decoder.h: the plan of a ragged batch (pages,
 * positions and slots from request lengths), the norm and position rotation of
 * queries and keys, attention with sinks, and the sampling of the next token.
 * Implemented in liblcml_fp8.so; the conventions of lcml_fp8.h hold: device
 * pointers, 64-bit sizes, a stream; asynchronous; no allocation; an lcml_status
 * with a message in lcml_last_error(), arguments checked before any work is
 * enqueued; no traps. Nothing reads device memory on the host, so every call can
 * be captured in a CUDA graph. The reference (LuisaML) has no counterpart of
 * these operators.
 */
#ifndef LCML_DECODE_STEP_H
#define LCML_DECODE_STEP_H

#include "lcml_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The plan of a step: row b of the batch holds held[b] tokens and brings
 * new_tokens[b] more.
 *   ended[b] (optional): the row's request is over. Its pages (the table's
 *       entries 0 .. ceil(held[b] / page_size) - 1, entries below 0 left out) go
 *       onto the free list in the order of rows and columns and become -1 in the
 *       table; the row then holds nothing, and new_tokens[b] is a new request's.
 *       Nothing counts who else holds a page: one that two rows share is given back
 *       by each that ends.
 *   start[b]  = ended[b] ? 0 : held[b]
 *   kv_len[b] = start[b] + new_tokens[b]
 *   cu_tokens = exclusive sums of new_tokens
 *   block_table: columns ceil(start / page_size) .. ceil(kv_len / page_size) - 1 of
 *       the rows, in order, take pages from the end of the free list
 *   positions[cu_tokens[b] + i] = start[b] + i
 *   slots[cu_tokens[b] + i]     = page * page_size + positions % page_size
 * so that start and kv_len are the lengths of lcml_kv_cache_write and
 * lcml_kv_attention. Packed tokens past cu_tokens[batch] get -1 in both maps.
 * kv_len may be held and free_count_out may be free_count: a captured step then
 * moves on with every replay.
 *
 * What does not fit shows in the device error word (lcml_device_error) and is
 * never followed: 8: the free list ran out; the entries left over are -1, and so
 * are their tokens' slots. 7: a negative length (taken as 0), tokens beyond
 * total_tokens (left out: cu_tokens[batch] <= total_tokens), a row longer than
 * the table's columns (-1 for those tokens' slots), or a free list that is
 * shorter than 0 or full (pages beyond free_capacity are dropped).
 */
typedef struct lcml_kv_plan_desc {
    int32_t batch;             /* <= 16384 */
    int32_t page_size;         /* <= 65536 */
    int32_t table_cols;        /* batch * table_cols <= 2^31 - 65537 */
    int64_t table_stride;
    int32_t *block_table;      /* device [batch, table_cols], changed in place */
    const int32_t *new_tokens; /* device [batch] */
    const int32_t *held;       /* device [batch] */
    const uint8_t *ended;      /* device [batch], 0 or not; optional */
    int32_t *free_pages;       /* device [free_capacity]: the free list, changed in place */
    int64_t free_capacity;
    const int32_t *free_count; /* device [1]: its pages are free_pages[0 .. free_count - 1] */
    int64_t total_tokens;      /* length of positions and slots */
    int32_t *cu_tokens;        /* device [batch + 1] */
    int32_t *start, *kv_len;   /* device [batch] */
    int32_t *positions, *slots; /* device [total_tokens] */
    int32_t *free_count_out;   /* device [1] */
} lcml_kv_plan_desc;

int lcml_kv_plan(const lcml_kv_plan_desc *desc, lcml_stream_t stream);

#define LCML_DTYPE_DOUBLE 11 /* ONNX's number; of inv_freq alone */

/*
 * Norm of every head of the queries and keys, then the rotation by position:
 *   y = x * weight / sqrt(mean(x^2) + eps)     (weight NULL: y = x)
 *   (a, b) -> (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i]
 * for the rotary / 2 pairs i of y's first `rotary` elements: (i, i + rotary / 2), or
 * (2 i, 2 i + 1) where `interleaved`. The rest of the head is only normed. fp32
 * inside, angles in 64 bits, rounded once to the type. A token of negative
 * position is not touched. Outputs may be the inputs themselves (same pointer and
 * strides) and do not overlap them otherwise.
 */
typedef struct lcml_qk_norm_rope_desc {
    int64_t tokens;
    int32_t q_heads, k_heads;  /* 0 .. 2^31 - 65537 */
    int32_t head_dim;          /* even, <= 512 */
    int32_t rotary;            /* even, <= head_dim */
    int dtype;                 /* FLOAT, FLOAT16 or BFLOAT16 */
    int interleaved;
    const void *q, *k;         /* [tokens, heads, head_dim], strides in elements */
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
    void *q_out, *k_out;       /* rows that do not overlap */
    int64_t q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride;
    const void *q_weight, *k_weight; /* [head_dim], optional */
    int weight_dtype;          /* dtype or FLOAT */
    float eps;
    const int32_t *positions;  /* device [tokens] */
    const void *inv_freq;      /* device [rotary / 2], radians per position */
    int inv_freq_dtype;        /* FLOAT or LCML_DTYPE_DOUBLE */
} lcml_qk_norm_rope_desc;

int lcml_qk_norm_rope(const lcml_qk_norm_rope_desc *desc, lcml_stream_t stream);

/*
 * lcml_kv_attention where the first `sinks` positions stay visible behind the
 * window: a query at position p sees the j <= p with j > p - window or j < sinks.
 * Pages between the sinks and the window are not looked at: their table entries
 * may be anything. sinks = 0, or window = 0: lcml_kv_attention as it is.
 * The workspace is the one of lcml_kv_attention_workspace_size(desc).
 */
int lcml_kv_attention_sinks(const lcml_kv_attention_desc *desc, int32_t sinks, lcml_stream_t stream);

/*
 * Draws a token of every row of logits. With x a row's logits and m their maximum,
 *   w_i = exp((x_i - m) / temperature)          (0 for a logit of -infinity)
 * and the order of the tokens by falling x (equal ones by rising index), the draw is
 * among the tokens that all of these keep:
 *   top_k: the first top_k (<= 0: all)
 *   top_p: of what top_k keeps, the fewest first ones whose w sum to at least top_p
 *          of its sum (>= 1 or NaN: all; at least one token stays)
 *   min_p: those with w_i >= min_p (<= 0 or NaN: all; above 1: as 1)
 * Token: the lowest index at which the kept tokens' w, summed by rising index,
 * passes uniform times their sum (uniform in [0, 1); outside it, the first or last
 * one). logprob: log of the token's share of that sum. temperature <= 0 or NaN: the
 * lowest index of the largest logit, logprob 0. A NaN logit counts as -infinity; a
 * row with +infinity gives the first of those, logprob 0; a row of -infinity alone
 * gives token -1 and logprob NaN.
 * Weights and sums are held in 64 bits, a weight good to 1e-12 of itself, but where up
 * to 256 tokens stay, to 2^-52 of the largest (a lighter one counts as that much). w below
 * 2^-1000 are 0. Equal calls give equal tokens. The same row in another batch or at
 * another alignment is summed in another order: there a token may differ whose border
 * uniform meets to the rounding of a 64-bit sum. Parameters are device arrays of one value
 * a row; NULL: off (temperature: 1).
 */
typedef struct lcml_sample_desc {
    int64_t rows, vocab;       /* vocab <= 2^31 - 65537 */
    const void *logits;        /* [rows, vocab], row stride ld elements */
    int64_t ld;
    int dtype;                 /* FLOAT, FLOAT16 or BFLOAT16 */
    const float *uniform;      /* device [rows] */
    const float *temperature;  /* device [rows] each, optional */
    const int32_t *top_k;
    const float *top_p, *min_p;
    int32_t *tokens;           /* device [rows] */
    float *logprob;            /* device [rows], optional */
} lcml_sample_desc;

int lcml_sample(const lcml_sample_desc *desc, lcml_stream_t stream);

#ifdef __cplusplus
}/* extern "C" */
#endif

#endif /* LCML_DECODE_STEP_H */
