// Norm of every head of the queries and keys and the rotation by position, in
// one pass (lcml_qk_norm_rope).
//
// A head lies in the registers of a few lanes: a lane takes chunks of E pairs
// (p, q), so a rotation needs no exchange, whichever way the pairs lie. Elements
// past the rotated ones are chunks that are only normed. A warp takes one token (or
// a share of its heads) and keeps the products of its cosines, sines and weights in
// registers from head to head; its lanes compute the cosines together. With the
// norm's factor r a pair costs r p, r q and four products, two elements at a time.
//
// The angle is reduced in 64 bits: position * (inv_freq / 2 pi) turns, less the
// nearest whole number, an error of 2^-53 of the turns (2^-30 of a turn at
// position 10^7); sincospi() of the rest rounds to fp32.
//
// Bound: HBM, every element read and written once. The heads come through a ring of
// four groups per warp in shared memory, as an output may be its input: loads
// into registers ahead of the stores left too few bytes on their way (8191 tokens of
// 32 + 8 heads of 128, bf16: 46.6 us loading as it goes, 39.3 one group ahead in
// registers, 32.5 so: 5.2 of a copy's 6.5 TB/s). Below some thousand tokens it is
// latency: position, angles (fp64), the first heads; one token 2.9 us, 3001 of
// 24 heads of 96 in fp32 14.2 us (16.4 where neighbouring pairs of a quarter turn: both
// kinds of chunk share a warp), floor 8.5. Heads that are not 16-byte aligned go element by
// element (E = 1): 8191 tokens of 40 heads 93 us, one 2.8.
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
    float eps, inv_dim;
    bool w_f32, freq_f64;
    int shares;  // warps a token
    int lanes;   // per head
};

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
__global__ void __launch_bounds__(kWarps * 32, E == 1 ? 2 : 3) k_qk_norm_rope(RopeArgs a) {
    // A lane's chunks of the next kAhead groups of heads, loaded by itself (E > 1).
    constexpr int kAhead = E == 1 ? 1 : 4 / C;
    __shared__ uint4 ring[E == 1 ? 1 : kWarps][kAhead][2 * C][E == 1 ? 1 : 32];
    __shared__ float2 turned[kWarps][256];
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    const int64_t token = item / a.shares;
    const int share = static_cast<int>(item - token * a.shares);
    const int half = a.rotary / 2, pairs = a.dim / 2;
    const int in_head = lane & (a.lanes - 1), in_warp = lane / a.lanes, per_warp = 32 / a.lanes;
    // where the chunks' elements lie
    int at[C][2];
    bool live[C], turn[C];
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
    }
    griddep_wait();
    if (token >= a.tokens) return;
    const int pos = __ldg(a.positions + token);
    if (pos < 0) return;

    // Heads go through the warp in groups, those of the queries first.
    const int q_groups = (a.heads[0] + per_warp - 1) / per_warp, groups = q_groups + (a.heads[1] + per_warp - 1) / per_warp;
    auto head_of = [&](int g, int &kind) {  // -1: none
        kind = g >= q_groups;
        const int head = (g - (kind ? q_groups : 0)) * per_warp + in_warp;
        return g < groups && head < a.heads[kind] ? head : -1;
    };
    auto fetch = [&](int g, int stage) {
        int kind;
        const int head = head_of(g, kind);
        const T *x = static_cast<const T *>(a.x[kind]) + token * a.xt[kind] + head * a.xh[kind];
        if (head >= 0) {
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (live[j])
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&ring[warp][stage][2 * j + h][lane])), "l"(x + at[j][h]) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (E > 1) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (!live[j]) ring[warp][i][2 * j][lane] = ring[warp][i][2 * j + 1][lane] = make_uint4(0, 0, 0, 0);
            if (i + 1 < kAhead) fetch(share + i * a.shares, i);
        }
    }

    // cosines and sines of the token's pairs
    for (int i = lane; i < half; i += 32) {
        const double f = a.freq_f64 ? __ldg(static_cast<const double *>(a.inv_freq) + i) : static_cast<double>(__ldg(static_cast<const float *>(a.inv_freq) + i));
        const double turns = pos * (f * 0.15915494309189533576888);
        float s, c;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
        turned[warp][i] = make_float2(c, s);
    }
    __syncwarp();
    // of a pair (p, q) with weights: p' = p c1 - q s1, q' = q c2 + p s2
    float c1[C][E], s1[C][E], c2[C][E], s2[C][E];
    int weights_of = -1;
    int stage = 0;
#pragma unroll 1
    for (int g = share; g < groups; g += a.shares) {
        if constexpr (E > 1) {
            fetch(g + (kAhead - 1) * a.shares, (stage + kAhead - 1) % kAhead);
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        }
        int kind;
        const int head = head_of(g, kind);
        const bool norm = a.w[kind] != nullptr;
        if (kind != weights_of) {
            weights_of = kind;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                float w[2 * E];
#pragma unroll
                for (int e = 0; e < 2 * E; ++e) w[e] = 1.0f;
                if (norm && live[j]) {
                    load_weight<T, E>(a.w[kind], a.w_f32, at[j][0], w);
                    load_weight<T, E>(a.w[kind], a.w_f32, at[j][1], w + E);
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float2 t = turn[j] ? turned[warp][(in_head + j * a.lanes) * E + e] : make_float2(1.0f, 0.0f);
                    const float wp = w[INTER ? 2 * e : e], wq = w[INTER ? 2 * e + 1 : E + e];
                    c1[j][e] = wp * t.x;
                    s1[j][e] = -wq * t.y;
                    c2[j][e] = wq * t.x;
                    s2[j][e] = wp * t.y;
                }
            }
        }
        float v[C][2 * E], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            if constexpr (E == 1) {
                const T *x = static_cast<const T *>(a.x[kind]) + token * a.xt[kind] + head * a.xh[kind];
#pragma unroll
                for (int h = 0; h < 2; ++h) v[j][h] = head >= 0 && live[j] ? Elem<T>::load(x + at[j][h]) : 0.0f;
            } else {
                load_vec<T, E, false>(reinterpret_cast<const T *>(&ring[warp][stage][2 * j][lane]), v[j]);
                load_vec<T, E, false>(reinterpret_cast<const T *>(&ring[warp][stage][2 * j + 1][lane]), v[j] + E);
            }
            float s0 = 0.0f, t0 = 0.0f;
#pragma unroll
            for (int e = 0; e < 2 * E; e += 2) fma2(s0, t0, v[j][e], v[j][e + 1], v[j][e], v[j][e + 1], s0, t0);
            sum += s0 + t0;
        }
        stage = (stage + 1) % kAhead;
        float r = 1.0f;
        if (norm) {
            for (int o = a.lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
        }
        if (head < 0) continue;
        T *y = static_cast<T *>(a.y[kind]) + token * a.yt[kind] + head * a.yh[kind];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            if (!live[j]) continue;
#pragma unroll
            for (int e = 0; e < 2 * E; e += 2) mul2(v[j][e], v[j][e + 1], v[j][e], v[j][e + 1], r, r);
            float o[2 * E];
            if (turn[j]) {
                if constexpr (E == 1 || INTER) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float p = v[j][INTER ? 2 * e : e], q = v[j][INTER ? 2 * e + 1 : E + e];
                        o[INTER ? 2 * e : e] = fmaf(q, s1[j][e], p * c1[j][e]);
                        o[INTER ? 2 * e + 1 : E + e] = fmaf(p, s2[j][e], q * c2[j][e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        mul2(o[e], o[e + 1], v[j][e], v[j][e + 1], c1[j][e], c1[j][e + 1]);
                        fma2(o[e], o[e + 1], v[j][E + e], v[j][E + e + 1], s1[j][e], s1[j][e + 1], o[e], o[e + 1]);
                        mul2(o[E + e], o[E + e + 1], v[j][E + e], v[j][E + e + 1], c2[j][e], c2[j][e + 1]);
                        fma2(o[E + e], o[E + e + 1], v[j][e], v[j][e + 1], s2[j][e], s2[j][e + 1], o[E + e], o[E + e + 1]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[INTER ? 2 * e : e] = v[j][INTER ? 2 * e : e] * c1[j][e];
                    o[INTER ? 2 * e + 1 : E + e] = v[j][INTER ? 2 * e + 1 : E + e] * c2[j][e];
                }
            }
            store_vec<T, E>(y + at[j][0], o);
            store_vec<T, E>(y + at[j][1], o + E);
        }
    }
}

template <typename T, int E, int C>
int launch_rope(RopeArgs a, bool inter, cudaStream_t st) {
    const int chunks = (a.dim / 2 + E - 1) / E;
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes * C < chunks) a.lanes *= 2;
    // A warp per token where there are 24 an SM, as many as it holds; else a token's heads are
    // shared until there are (one token of 40 heads of 128: one warp 8 us, ten 2.9; 300 tokens:
    // four warps each 5.9, all ten 4.3; 3001 of 24 heads of 96 in fp32: one 20.4, two 16.6). The
    // share is rounded up, which may leave a few warps to a second round: 1000 of 40 heads get four, 9.1
    // us, where three, all at once, take 7.4.
    const int per_warp = 32 / a.lanes;
    const int64_t most = (a.heads[0] + per_warp - 1) / per_warp + (a.heads[1] + per_warp - 1) / per_warp;
    const int64_t want = static_cast<int64_t>(sm_count()) * 24;
    int64_t shares = (want + a.tokens - 1) / a.tokens;
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
    // heads are counted in 32 bits, a group of up to 32 at a time
    LCML_CHECK_ARG(d->q_heads <= 0x7fffffff - 65536 && d->k_heads <= 0x7fffffff - 65536, "lcml_qk_norm_rope: too many heads");
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
               1.0f / static_cast<float>(d->head_dim),
               d->weight_dtype == LCML_DTYPE_FLOAT,
               d->inv_freq_dtype == LCML_DTYPE_DOUBLE,
               1,
               1};
    cudaStream_t st = to_cuda(stream);
    if (d->dtype == LCML_DTYPE_FLOAT) return dispatch_rope<float>(a, d->interleaved != 0, st);
    if (d->dtype == LCML_DTYPE_FLOAT16) return dispatch_rope<__half>(a, d->interleaved != 0, st);
    return dispatch_rope<__nv_bfloat16>(a, d->interleaved != 0, st);
}
