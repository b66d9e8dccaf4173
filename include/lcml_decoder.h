/*
 * lcml_decoder.h — C ABI of the operators around the FP8 GEMMs of a decoder
 * layer: RMS norm with the residual's addition and an e4m3 output, the paged
 * e4m3 key/value cache (quantizing write, read back) and the attention over
 * it. Implemented in liblcml_fp8.so; the conventions of lcml_fp8.h hold:
 * device pointers, 64-bit sizes, a stream; asynchronous; no allocation; an
 * lcml_status with a message in lcml_last_error(), arguments checked before
 * any work is enqueued; no traps. The reference (LuisaML) has no counterpart
 * of these operators.
 */
#ifndef LCML_DECODER_H
#define LCML_DECODER_H

#include "lcml_fp8.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * RMS norm with the residual's addition and an e4m3 output:
 *   h = x + residual            (fp32; residual may be NULL: h = x)
 *   y = h * w * 1 / sqrt(mean(h^2) + eps)
 *   s = max|y| / 448 per row (1 for an all-zero row; NaN ignored), written to
 *       scale_out [rows]; or, with `scale` (device, one float), s = *scale
 *   q = e4m3(y / s)             (QuantizeLinear; y / s computed as h * w *
 *       (1 / sqrt(..) / s), the codec by the rule of the GEMM's epilogues)
 * q and scale_out are the A operand and scale_a (LCML_SCALE_ROW, or TENSOR
 * for a given scale) of lcml_fp8_gemm. The norm is taken of the fp32 sum;
 * h_out receives it rounded to x's type (may alias x or residual; NULL: not
 * written). Exactly one of scale and scale_out is given.
 */
typedef struct lcml_rmsnorm_desc {
    int64_t rows, cols;
    const void *x;         /* [rows, cols], row stride ldx elements */
    int64_t ldx;
    const void *residual;  /* optional, x's type, row stride ldr */
    int64_t ldr;
    void *h_out;           /* optional, x's type, row stride ldh */
    int64_t ldh;
    const void *weight;    /* [cols] */
    int x_dtype;           /* FLOAT, FLOAT16 or BFLOAT16 */
    int weight_dtype;      /* x_dtype or FLOAT */
    float eps;
    const float *scale;    /* device [1]: a calibrated output scale */
    float *scale_out;      /* device [rows]: receives the dynamic scales */
    uint8_t *q;            /* [rows, cols] e4m3, dense */
} lcml_rmsnorm_desc;

int lcml_rmsnorm_quantize(const lcml_rmsnorm_desc *desc, lcml_stream_t stream);

/*
 * Paged e4m3 key/value cache. Page p holds page_size tokens of every head:
 *   k, v             [num_pages, kv_heads, page_size, head_dim] e4m3
 *   k_scale, v_scale [num_pages, kv_heads, page_size / scale_block] fp32
 * so a value is decode(code) * the scale of its block of scale_block tokens.
 * head_dim: 64, 128 or 256; scale_block: a multiple of 16 that divides
 * page_size, with scale_block * head_dim <= 32768. k and v are 16-byte
 * aligned; scales are finite and not negative, as lcml_kv_cache_write leaves
 * them. kv_heads <= 4096, page_size <= 65536 and num_pages * kv_heads *
 * page_size < 2^31 (a row of head_dim codes has a 32-bit index, an address 64
 * bits).
 */
typedef struct lcml_kv_cache {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int64_t num_pages;
    int32_t page_size, kv_heads, head_dim, scale_block;
} lcml_kv_cache;

/*
 * A ragged batch: sequence b owns tokens cu_tokens[b] .. cu_tokens[b + 1] - 1
 * of the packed token dimension (cu_tokens[0] >= 0, more where the call takes a
 * part of a longer batch; cu_tokens[batch] <= total_tokens), and position t of
 * sequence b lives in slot t % page_size of page
 * block_table[b * table_stride + t / page_size]; cu_tokens does not
 * decrease. A table entry outside [0, num_pages), or a position past the
 * table's columns, is never followed: a write or read skips it, attention
 * leaves its tokens out (what it returns for that sequence means nothing), and
 * the device error word (lcml_device_error) gets code 6. A negative length sets
 * it to 7: a write or read skips the sequence's tokens, to attention it holds none.
 */
typedef struct lcml_kv_batch {
    int32_t batch;
    int32_t table_cols;          /* columns (pages per sequence) of block_table */
    const int32_t *block_table;  /* device [batch, table_cols] */
    int64_t table_stride;
    const int32_t *cu_tokens;    /* device [batch + 1] */
    const int32_t *lengths;      /* device [batch]: see each function */
    int64_t total_tokens;
} lcml_kv_batch;

/*
 * Quantizes new tokens into the cache. Sequence b's tokens take the positions
 * lengths[b], lengths[b] + 1, ...: lengths[b] is the number of tokens it
 * already holds. Per block of scale_block positions and head:
 *   s = max(s_old, max|x| / 448 over the block's new values)
 * with s_old the stored scale if the block holds earlier tokens (else 0);
 * max|x| takes finite values only, a nonzero s is at least 2^-100, and an
 * all-zero block keeps s = 0 and codes 0. New codes are e4m3(x / s) (an
 * infinity saturates, NaN stays NaN). Where s > s_old the block's earlier
 * codes are re-encoded, e4m3(decode(code) * s_old / s). Slots after the new
 * tokens are left alone. Two sequences of one call must not write one page.
 * k, v: [total_tokens, kv_heads, head_dim] with token and head strides in
 * elements, FLOAT, FLOAT16 or BFLOAT16.
 */
int lcml_kv_cache_write(const lcml_kv_cache *cache, const lcml_kv_batch *batch, const void *k, int64_t k_token_stride,
                        int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                        lcml_stream_t stream);

/*
 * Reads tokens back: token cu_tokens[b] + i of k and v receives position
 * lengths[b] + i of sequence b, decode(code) * scale rounded once to dtype.
 * k, v: dense [total_tokens, kv_heads, head_dim], 16-byte aligned; either may
 * be NULL.
 */
int lcml_kv_cache_read(const lcml_kv_cache *cache, const lcml_kv_batch *batch, void *k, void *v, int dtype,
                       lcml_stream_t stream);

/*
 * Attention over the cache. Sequence b holds lengths[b] tokens (the new ones
 * written already); its n = cu_tokens[b + 1] - cu_tokens[b] queries are the
 * last n of them: query i has position lengths[b] - n + i and sees the
 * positions j <= its own (causal = 0: all j < lengths[b]), with window > 0
 * only those with j > position - window. Query head h reads cache head
 * h / (q_heads / kv_heads).
 *   x_j = softmax_scale * q . k_j;  softcap > 0: x_j = softcap * tanh(x_j / softcap)
 *   out = sum_j softmax(x)_j v_j,   lse = log sum_j exp(x_j)
 * A query that sees nothing gets zeros and lse -inf. Scores, the softmax's
 * maximum and sum, and the output accumulate in fp32. The softmax's weights enter
 * the product with the values as halves (11 significant bits: FLOAT16 outputs
 * measured 2.9e-4 off, 2.1e-4 of it their own rounding), q as it is or, on the
 * tensor-core path, as a sum of e4m3 parts: exact for elements above 2^-9
 * (BFLOAT16) or 2^-6 (FLOAT16) of the row's largest, within 2^-17 of that one
 * for smaller ones. A value block of scale 0 counts in the sum alone. What the
 * masked slots hold (NaN codes included) does not matter.
 * max_tokens: an upper bound of the n (host side). It and the extents pick the
 * kernels: the closer it is, the fewer launches (exact for a batch of equal
 * lengths). Where total_tokens is padded, the padded total picks, and every
 * query is computed. A sequence with more queries, or longer than its block
 * table reaches, is not computed in full and sets the device error word to 7.
 * workspace: lcml_kv_attention_workspace_size(desc) bytes, 16-byte aligned,
 * contents on entry do not matter (NULL when the size is 0).
 */
typedef struct lcml_kv_attention_desc {
    const lcml_kv_cache *cache;
    const lcml_kv_batch *batch;
    const void *q;            /* [total_tokens, q_heads, head_dim], strides in elements */
    int64_t q_token_stride, q_head_stride;
    void *out;                /* same shape and type, rows that do not overlap */
    int64_t out_token_stride, out_head_stride;
    float *lse;               /* optional, dense [total_tokens, q_heads] */
    int32_t q_heads;
    int dtype;                /* FLOAT16 or BFLOAT16 */
    int64_t max_tokens;
    float softmax_scale;
    float softcap;            /* 0: none */
    int32_t window;           /* 0: none */
    int causal;
    void *workspace;
    /* Kernel choice, per call (0 = automatic): 1 the streaming kernel for
     * every sequence, 2 the tensor-core kernel for every sequence (head_dim
     * 64 or 128). For cross-checking and tuning. */
    int variant;
} lcml_kv_attention_desc;

int64_t lcml_kv_attention_workspace_size(const lcml_kv_attention_desc *desc); /* -1 on a bad desc */
int lcml_kv_attention(const lcml_kv_attention_desc *desc, lcml_stream_t stream);

#ifdef __cplusplus
}/* extern "C" */
#endif

#endif /* LCML_DECODER_H */
