// What the two attention kernels (kv_attention.cu, kv_attention_tc.cu) share.
#pragma once

#include "lcml_decoder.cuh"

namespace lcml {

struct AttnArgs {
    lcml_kv_cache c;
    lcml_kv_batch b;
    const void *q;
    void *out;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    float *lse;
    int group;         // q_heads / kv_heads
    int bf16;          // type of q and out
    float scale_log2;  // softmax_scale * log2(e)
    float cap, inv_cap;  // tanh cap in units of the plain score, 0: none; softmax_scale / cap
    int window, causal;
    int64_t max_tokens;
    int *err;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Score in log2 units: x = q . k softmax_scale, capped, times log2(e).
// tanh(t) = 1 - 2 / (e^2t + 1): its error (a few fp32 ulps of 1, times cap)
// is far below that of tanh.approx, whose 2^-11 would shift a score by
// cap / 2048. Saturates to +-1 for large |t|; NaN stays NaN.
__device__ __forceinline__ float cap_score(float dot, float inv_cap, float cap) {
    const float t = dot * inv_cap;
    const float e = exp2_approx(t * (2.0f * kLog2e));
    return cap * kLog2e * (1.0f - __fdividef(2.0f, e + 1.0f));
}

// The scale of a block of values takes part in the softmax's exponent: with
// a_j = x_j + log2(s_j) the weights 2^(a_j - m) multiply codes, and the sum
// takes 2^(a_j - m) / s_j. A scale below 2^-100 (an all-zero block, whose codes
// are zero) counts as 1.
__device__ __forceinline__ float value_scale(float s) { return s >= 7.888609052210118e-31f ? s : 1.0f; }

// Two e4m3 codes -> two halves (exact), low byte first.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t b) {
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(b));
    return h;
}

// The four codes of a word -> two pairs of halves.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// The tensor-core path for long runs of queries (kv_attention_tc.cu).
bool kv_attention_tc_fits(const lcml_kv_attention_desc *d);
int kv_attention_tc(const lcml_kv_attention_desc *d, const AttnArgs &a, int min_rows, cudaStream_t st);

}// namespace lcml
