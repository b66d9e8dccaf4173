// Norm of every head of the queries and keys and the rotation by position, in
// one pass (lcml_qk_norm_rope).
//
// A head lies in the registers of a few lanes: a lane takes chunks of E pairs
// (a, b), so a rotation needs no exchange, whichever way the pairs lie. Elements
// past the rotated ones are chunks that are only normed. A warp takes one token (or a
// share of its heads) and keeps its cosines, sines and weights in registers from
// head to head; its lanes compute the cosines together, one pair each.
//
// The angle is reduced in 64 bits: position * (inv_freq / 2 pi) turns, less the
// nearest whole number, an error of 2^-53 of the turns (2^-30 of a turn at
// position 10^7); sincospif() of the rest rounds to fp32.
//
// Bound: HBM, every element read and written once.
#include "lcml_decoder.cuh"

#include "../../include/lcml_decode_step.h"

namespace lcml {
namespace {

constexpr int kWarps = 8;  // per CTA

struct RopeArgs {
    const void *x[2];
    void *y[2];
    int64_t xt[2], xh[2], yt[2], yh[2];
    int heads[2];
    const void *w[2];
    const int32_t *positions;
    const void *inv_freq;
    int64_t tokens;
    int dim, rotary;
    float eps;
    bool w_f32, freq_f64;
    int shares;  // warps a token
    int lanes;   // per head
};

// E elements at p, or one by one where E is 1.
template <typename T, int E>
__device__ __forceinline__ void load_part(const void *base, int64_t at, float *v) {
    load_vec<T, E, false>(static_cast<const T *>(base) + at, v);
}

template <typename T, int E>
__device__ __forceinline__ void load_weight(const void *base, bool f32, int64_t at, float *v) {
    if (f32) {
        const float *p = static_cast<const float *>(base) + at;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = __ldg(p + e);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = Elem<T>::load(static_cast<const T *>(base) + at + e);
    }
}

// E pairs per chunk, C chunks per lane.
template <typename T, int E, int C, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) k_qk_norm_rope(RopeArgs a) {
    __shared__ float2 turned[kWarps][256];
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    const int64_t token = item / a.shares;
    const int share = static_cast<int>(item % a.shares);
    griddep_wait();
    if (token >= a.tokens) return;
    const int pos = __ldg(a.positions + token);
    if (pos < 0) return;

    // cosines and sines of the token's pairs
    const int half = a.rotary / 2, pairs = a.dim / 2;
    for (int i = lane; i < half; i += 32) {
        const double f = a.freq_f64 ? __ldg(static_cast<const double *>(a.inv_freq) + i) : static_cast<double>(__ldg(static_cast<const float *>(a.inv_freq) + i));
        const double turns = pos * (f * 0.15915494309189533576888);
        float s, c;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
        turned[warp][i] = make_float2(c, s);
    }
    __syncwarp();

    const int in_head = lane % a.lanes, per_warp = 32 / a.lanes;
    // where the chunks' elements lie, and their cosines and sines
    int at[C][2];
    bool live[C], turn[C];
    float cs[C][E], sn[C][E];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int p = (in_head + j * a.lanes) * E;  // the chunk's first pair
        live[j] = p < pairs;
        turn[j] = p < half;
        if (INTER) {
            at[j][0] = 2 * p;
            at[j][1] = 2 * p + E;
        } else if (p < half) {
            at[j][0] = p;
            at[j][1] = p + half;
        } else {
            at[j][0] = p + half;  // 2 half + (p - half)
            at[j][1] = p + pairs;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 t = turn[j] ? turned[warp][p + e] : make_float2(1.0f, 0.0f);
            cs[j][e] = t.x;
            sn[j][e] = t.y;
        }
    }
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
        const int heads = a.heads[kind];
        const T *x = static_cast<const T *>(a.x[kind]) + token * a.xt[kind];
        T *y = static_cast<T *>(a.y[kind]) + token * a.yt[kind];
        const bool norm = a.w[kind] != nullptr;
        float w[C][2 * E];
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (norm && live[j]) load_weight<T, E>(a.w[kind], a.w_f32, at[j][h], w[j] + h * E);
                else
#pragma unroll
                    for (int e = 0; e < E; ++e) w[j][h * E + e] = 1.0f;
            }
        for (int h0 = share * per_warp; h0 < heads; h0 += a.shares * per_warp) {
            const int head = h0 + lane / a.lanes;
            const bool on = head < heads && lane < per_warp * a.lanes;
            float v[C][2 * E];
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < C; ++j) {
#pragma unroll
                for (int e = 0; e < 2 * E; ++e) v[j][e] = 0.0f;
                if (on && live[j]) {
                    load_part<T, E>(x, head * a.xh[kind] + at[j][0], v[j]);
                    load_part<T, E>(x, head * a.xh[kind] + at[j][1], v[j] + E);
                }
            }
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
                for (int e = 0; e < 2 * E; ++e) sum = fmaf(v[j][e], v[j][e], sum);
            for (int o = a.lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float r = norm ? rsqrtf(sum / static_cast<float>(a.dim) + a.eps) : 1.0f;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                if (!on || !live[j]) continue;
#pragma unroll
                for (int e = 0; e < 2 * E; ++e) v[j][e] *= r * w[j][e];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float &p = v[j][INTER ? 2 * e : e], &q = v[j][INTER ? 2 * e + 1 : E + e];
                    const float t = p * cs[j][e] - q * sn[j][e], u = q * cs[j][e] + p * sn[j][e];
                    p = turn[j] ? t : p;
                    q = turn[j] ? u : q;
                }
                store_vec<T, E>(y + head * a.yh[kind] + at[j][0], v[j]);
                store_vec<T, E>(y + head * a.yh[kind] + at[j][1], v[j] + E);
            }
        }
    }
}

template <typename T, int E, int C>
int launch_rope(RopeArgs a, bool inter, cudaStream_t st) {
    const int chunks = (a.dim / 2 + E - 1) / E;
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes * C < chunks) a.lanes *= 2;
    // A warp per token where there are enough of them; else its heads are shared.
    const int per_warp = 32 / a.lanes;
    const int most = (max(a.heads[0], a.heads[1]) + per_warp - 1) / per_warp;
    const int64_t want = static_cast<int64_t>(sm_count()) * 4 * kWarps;
    int64_t shares = want / a.tokens;
    shares = shares < 1 ? 1 : (shares > most ? most : shares);
    a.shares = static_cast<int>(shares);
    const int64_t grid = (a.tokens * shares + kWarps - 1) / kWarps;
    LCML_CHECK_ARG(grid <= 0x7fffffff, "lcml_qk_norm_rope: too many tokens for one call");
    return launch_dependent(inter ? k_qk_norm_rope<T, E, C, true> : k_qk_norm_rope<T, E, C, false>, dim3(static_cast<unsigned>(grid)), kWarps * 32, 0, st,
                            "qk_norm_rope", a);
}

template <typename T>
int dispatch_rope(const RopeArgs &a, bool inter, cudaStream_t st) {
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    bool fits = a.rotary % (2 * E) == 0 && a.dim % (2 * E) == 0;
    for (int i = 0; i < 2; ++i)
        fits = fits && (a.heads[i] == 0 || (aligned(a.x[i], 16) && aligned(a.y[i], 16) && a.xt[i] % E == 0 && a.xh[i] % E == 0 && a.yt[i] % E == 0 && a.yh[i] % E == 0));
    if (fits) {
        if constexpr (E == 4) {
            if (a.dim > 256) return launch_rope<T, E, 2>(a, inter, st);
        }
        return launch_rope<T, E, 1>(a, inter, st);
    }
    if (a.dim <= 128) return launch_rope<T, 1, 2>(a, inter, st);
    return launch_rope<T, 1, 8>(a, inter, st);
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" int lcml_qk_norm_rope(const lcml_qk_norm_rope_desc *d, lcml_stream_t stream) {
    LCML_CHECK_ARG(d != nullptr, "lcml_qk_norm_rope: null descriptor");
    LCML_CHECK_ARG(d->tokens >= 0 && d->q_heads >= 0 && d->k_heads >= 0, "lcml_qk_norm_rope: negative extent");
    LCML_CHECK_ARG(d->head_dim > 0 && d->head_dim % 2 == 0 && d->head_dim <= 512, "lcml_qk_norm_rope: head_dim %d is not even and at most 512", d->head_dim);
    LCML_CHECK_ARG(d->rotary >= 0 && d->rotary % 2 == 0 && d->rotary <= d->head_dim, "lcml_qk_norm_rope: rotary %d is not even and at most head_dim %d",
                   d->rotary, d->head_dim);
    LCML_CHECK_ARG(d->dtype == LCML_DTYPE_FLOAT || d->dtype == LCML_DTYPE_FLOAT16 || d->dtype == LCML_DTYPE_BFLOAT16, "lcml_qk_norm_rope: dtype %d unsupported",
                   d->dtype);
    LCML_CHECK_ARG(d->weight_dtype == d->dtype || d->weight_dtype == LCML_DTYPE_FLOAT || (!d->q_weight && !d->k_weight),
                   "lcml_qk_norm_rope: weight_dtype %d is neither dtype nor FLOAT", d->weight_dtype);
    LCML_CHECK_ARG(d->inv_freq_dtype == LCML_DTYPE_FLOAT || d->inv_freq_dtype == LCML_DTYPE_DOUBLE, "lcml_qk_norm_rope: inv_freq_dtype %d unsupported",
                   d->inv_freq_dtype);
    LCML_CHECK_ARG(d->eps >= 0.0f, "lcml_qk_norm_rope: eps is negative or NaN");
    if (d->tokens == 0 || d->q_heads + static_cast<int64_t>(d->k_heads) == 0) return LCML_OK;
    LCML_CHECK_ARG((d->q_heads == 0 || (d->q && d->q_out)) && (d->k_heads == 0 || (d->k && d->k_out)) && d->positions && (d->inv_freq || d->rotary == 0),
                   "lcml_qk_norm_rope: null pointer");
    const uintptr_t es = d->dtype == LCML_DTYPE_FLOAT ? 4 : 2, ws = d->weight_dtype == LCML_DTYPE_FLOAT ? 4 : 2;
    LCML_CHECK_ARG(aligned(d->q, es) && aligned(d->k, es) && aligned(d->q_out, es) && aligned(d->k_out, es) && aligned(d->q_weight, ws) && aligned(d->k_weight, ws) &&
                       aligned(d->positions, 4) && aligned(d->inv_freq, d->inv_freq_dtype == LCML_DTYPE_FLOAT ? 4 : 8),
                   "lcml_qk_norm_rope: a pointer is not aligned to its element size");
    const int64_t strides[8] = {d->q_token_stride, d->q_head_stride, d->k_token_stride, d->k_head_stride,
                                d->q_out_token_stride, d->q_out_head_stride, d->k_out_token_stride, d->k_out_head_stride};
    for (int64_t s : strides) LCML_CHECK_ARG(s >= 0, "lcml_qk_norm_rope: negative stride");
    for (int i = 0; i < 2; ++i) {  // rows of an output are written by different warps: either stride covers the rows of the other
        const int64_t ts = strides[4 + 2 * i], hs = strides[5 + 2 * i], heads = i ? d->k_heads : d->q_heads, dim = d->head_dim;
        LCML_CHECK_ARG(heads == 0 || ((d->tokens == 1 || ts >= dim) && (heads == 1 || hs >= dim) &&
                                      (d->tokens == 1 || heads == 1 || ts >= (heads - 1) * hs + dim || hs >= (d->tokens - 1) * ts + dim)),
                       "lcml_qk_norm_rope: rows of an output overlap (strides %lld and %lld)", (long long)ts, (long long)hs);
    }
    RopeArgs a{{d->q, d->k},
               {d->q_out, d->k_out},
               {strides[0], strides[2]},
               {strides[1], strides[3]},
               {strides[4], strides[6]},
               {strides[5], strides[7]},
               {d->q_heads, d->k_heads},
               {d->q_weight, d->k_weight},
               d->positions,
               d->inv_freq,
               d->tokens,
               d->head_dim,
               d->rotary,
               d->eps,
               d->weight_dtype == LCML_DTYPE_FLOAT,
               d->inv_freq_dtype == LCML_DTYPE_DOUBLE,
               1,
               1};
    cudaStream_t st = to_cuda(stream);
    if (d->dtype == LCML_DTYPE_FLOAT) return dispatch_rope<float>(a, d->interleaved != 0, st);
    if (d->dtype == LCML_DTYPE_FLOAT16) return dispatch_rope<__half>(a, d->interleaved != 0, st);
    return dispatch_rope<__nv_bfloat16>(a, d->interleaved != 0, st);
}
