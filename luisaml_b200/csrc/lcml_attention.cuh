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
// takes 2^(a_j - m) / s_j. A block of scale 0 adds nothing to the output but its
// share of the sum, so any scale small enough does: 2^-80 keeps its keys out of
// the reference maximum m (as 1 they would push the other weights by their
// scales, e.g. 2^-16 for values of 0.01, into subnormal halves), and its weights
// only flush to 0 (2^-126) below about 2^-46 of the largest weight times its
// scale. Scales below 2^-100 do not occur in a written cache and count as 0.
__device__ __forceinline__ float value_scale(float s) { return s >= 7.888609052210118e-31f ? s : 8.271806125530277e-25f; }

// The four codes of a word -> two pairs of halves (exact), low byte first.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// A row of q as e4m3 parts. Times 2^(7 - e) its largest element (exponent e)
// comes to [128, 256); part 1 is the nearest e4m3 value of that, part 2 the
// nearest of what is left, and so on. e4m3 has 4 significant bits and the rest
// has a sign, so two parts are a bf16 (8 bits) exactly and three an fp16 (11),
// but for elements whose last bit is below e4m3's least step (2^-9; those less
// than 2^-9, for fp16 2^-6, of the row's largest): an error of 2^-10, 2^-17 of the
// row's largest element. A row with an infinity
// or NaN becomes NaN.
template <int NP>
struct QScale {
    float up, factor;  // 2^(7 - e) and 2^(e - 7)
    bool special;
    // mx: the row's largest magnitude as bits of its type (16-bit floats order
    // like their bits, NaN above infinity)
    __device__ __forceinline__ explicit QScale(uint32_t mx) {
        const uint32_t top = NP == 2 ? mx << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(mx))));
        special = top >= 0x7f800000u;
        int e = static_cast<int>(top >> 23);
        e = top == 0 ? 127 : min(max(e, 8), 253);
        up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23) * 128.0f;
        factor = __uint_as_float(static_cast<uint32_t>(e) << 23) * 0.0078125f;
    }
};

// Four elements (two words of 16-bit floats) -> one word of each part.
template <int NP>
__device__ __forceinline__ void split_q(uint32_t w0, uint32_t w1, const QScale<NP> &s, uint32_t (&parts)[NP]) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? w0 : w1, bits = i & 1 ? w >> 16 : w & 0xffffu;
        x[i] = s.up * (NP == 2 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits))));
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const uint32_t c = cvt_e4m3x2(x[0], x[1]) | (cvt_e4m3x2(x[2], x[3]) << 16);
        parts[p] = s.special ? 0x7f7f7f7fu : c;
        if (p + 1 < NP) {
            float f[4];
            e4m3x2_decode(c & 0xffffu, f[0], f[1]);
            e4m3x2_decode(c >> 16, f[2], f[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] -= f[i];
        }
    }
}

constexpr int kTcBlockRows = 256;  // rows per CTA of the tensor-core kernel

// The tensor-core path for long runs of queries (kv_attention_tc.cu).
bool kv_attention_tc_fits(const lcml_kv_attention_desc *d);
int kv_attention_tc(const lcml_kv_attention_desc *d, const AttnArgs &a, int min_rows, cudaStream_t st);

}// namespace lcml
