// RMS norm with the residual's addition and an e4m3 output
// (lcml_rmsnorm_quantize).
//
// One CTA per row; the row stays in registers as h * w between the reduction
// and the quantization, so x and the residual are read once. With
//   y = h w r,  r = 1 / sqrt(mean(h^2) + eps) > 0,
// max|y| = r max|h w|, so the sum of squares and the maximum are reduced
// together: one block reduction per row, not two.
//
// Bound: HBM (x + residual + h + 1 byte per element) for many rows (8191 x 5000
// fp32: 41 us, 5.0 of a copy's 6.5 TB/s), the latency of one load, one block
// reduction and one store for few (1 x 4096: 2.0 us in a graph). Rows whose width
// or start does not divide by 4 elements go one element at a time: 2000 x 2157
// fp16 12.5 us in a graph, 2000 x 2156 5.5.
#include "lcml_decoder.cuh"

namespace lcml {
namespace {

struct NormArgs {
    int64_t cols, ldx, ldr, ldh;
    const void *x, *residual;
    void *h_out;
    const void *weight;
    float eps;
    const float *scale;
    float *scale_out;
    uint8_t *q;
};

// Block-wide (sum, max of values >= 0): every thread gets both.
__device__ __forceinline__ void block_sum_max(float &sum, float &mx) {
    __shared__ float red_s[32], red_m[32];
    auto warp_max = [](float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    mx = warp_max(mx);
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (nw == 1) return;
    if (l == 0) {
        red_s[w] = sum;
        red_m[w] = mx;
    }
    __syncthreads();
    sum = l < nw ? red_s[l] : 0.0f;
    mx = warp_max(l < nw ? red_m[l] : 0.0f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}

// r / s for r ~ 1 / sqrt(ms), rounded about once: one Newton step for r, whose
// correction c stays apart, then one for the quotient. All elements of a row share
// this factor's error: of 8191 x 5000 fp32 values 48 had another code than in 64
// bits without the steps, 33 have with them, 31 with the factor from 64 bits.
__device__ __forceinline__ float norm_factor(float r, float ms, float s) {
    const float u = r * ms, ue = fmaf(r, ms, -u);
    const float c = 0.5f * r * (fmaf(-u, r, 1.0f) - ue * r);
    const float inv = __frcp_rn(s), f = r * inv;
    return fmaf(inv, fmaf(-f, s, r) + c, f);
}

// E elements per access (E = 1: rows of any alignment), VPT accesses per
// thread: cols <= E * VPT * blockDim.x.
template <typename T, typename W, int E, int VPT>
__global__ void __launch_bounds__(1024) k_rmsnorm_quantize(NormArgs a) {
    griddep_launch_dependents();  // the GEMM behind may start its set-up
    const int64_t row = blockIdx.x;
    const int nv = static_cast<int>(a.cols / E);
    // A thread past the row's end reads the last access again and drops it:
    // loads and arithmetic without branches. What it reads may be h already,
    // where h_out is x or residual, so it counts neither in the sum nor in the
    // maximum; the owner's own load comes before its store.
    float v[VPT * E];
    griddep_wait();
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
#pragma unroll
    for (int j = 0; j < VPT; ++j) load_vec<T, E, false>(x + static_cast<int64_t>(min(static_cast<int>(threadIdx.x + j * blockDim.x), nv - 1)) * E, v + j * E);
    if (a.residual != nullptr) {
        const T *r = static_cast<const T *>(a.residual) + row * a.ldr;
        float t[VPT * E];
#pragma unroll
        for (int j = 0; j < VPT; ++j) load_vec<T, E, false>(r + static_cast<int64_t>(min(static_cast<int>(threadIdx.x + j * blockDim.x), nv - 1)) * E, t + j * E);
#pragma unroll
        for (int k = 0; k < VPT * E; ++k) v[k] += t[k];
    }
    if (a.h_out != nullptr) {
        T *h = static_cast<T *>(a.h_out) + row * a.ldh;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < nv) store_vec<T, E>(h + static_cast<int64_t>(i) * E, v + j * E);
        }
    }
    float sum = 0.0f, mx = 0.0f;  // fmaxf ignores NaN
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        float w[E];
        load_vec<W, E>(static_cast<const W *>(a.weight) + static_cast<int64_t>(min(i, nv - 1)) * E, w);
        float s0 = 0.0f, s1 = 0.0f, top = 0.0f;
        if constexpr (E == 1) {
            s0 = v[j] * v[j];
            v[j] *= w[0];
            top = fabsf(v[j]);
        } else {
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float &v0 = v[j * E + e], &v1 = v[j * E + e + 1];
                fma2(s0, s1, v0, v1, v0, v1, s0, s1);
                mul2(v0, v1, v0, v1, w[e], w[e + 1]);
                top = fmaxf(fmaxf(top, fabsf(v0)), fabsf(v1));
            }
        }
        sum += i < nv ? s0 + s1 : 0.0f;
        mx = fmaxf(mx, i < nv ? top : 0.0f);
    }
    block_sum_max(sum, mx);
    const float r = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
    const float s = a.scale != nullptr ? __ldg(a.scale) : scale_from_amax(mx * r);
    if (a.scale_out != nullptr && threadIdx.x == 0) a.scale_out[row] = s;
    // y / s as h w (r / s): one product per element, and the codec by the rule
    // of the fused GEMM epilogues (quantize_block_rcp). It differs from a
    // division only where y / s lies within a few fp32 ulps of an e4m3
    // boundary, as y itself is uncertain by the order of its sum.
    const float f = norm_factor(r, sum / static_cast<float>(a.cols) + a.eps, s);
    const bool ok = scale_fast_ok(s, f);
    uint8_t *q = a.q + row * a.cols;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        if (i < nv) {
            if constexpr (E == 1) {
                q[i] = static_cast<uint8_t>(ok ? quantize_rcp1(v[j], f) : quantize1(v[j] * r, s));
            } else {
                uint32_t c[E / 4];
                if (ok) {
                    quantize_block_rcp<E>(v + j * E, f, c);
                } else {
#pragma unroll
                    for (int k = 0; k < E / 4; ++k) {
                        c[k] = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[k] |= quantize1(v[j * E + k * 4 + e] * r, s) << (8 * e);
                    }
                }
                if constexpr (E == 8) *reinterpret_cast<uint2 *>(q + static_cast<int64_t>(i) * 8) = make_uint2(c[0], c[1]);
                else *reinterpret_cast<uint32_t *>(q + static_cast<int64_t>(i) * 4) = c[0];
            }
        }
    }
}

// Rows too long for the registers of one CTA: three passes over the row (the
// second and third mostly from L1 / L2). h_out may alias x or residual, so h
// is written in the last pass.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) k_rmsnorm_quantize_long(NormArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const T *rp = a.residual != nullptr ? static_cast<const T *>(a.residual) + row * a.ldr : nullptr;
    const W *w = static_cast<const W *>(a.weight);
    auto h = [&](int64_t c) { return Elem<T>::load(x + c) + (rp != nullptr ? Elem<T>::load(rp + c) : 0.0f); };
    float sum = 0.0f, mx = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float v = h(c);
        sum = fmaf(v, v, sum);
        mx = fmaxf(mx, fabsf(v * Elem<W>::load(w + c)));
    }
    block_sum_max(sum, mx);
    const float r = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
    const float s = a.scale != nullptr ? __ldg(a.scale) : scale_from_amax(mx * r);
    if (a.scale_out != nullptr && threadIdx.x == 0) a.scale_out[row] = s;
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float v = h(c);
        a.q[row * a.cols + c] = static_cast<uint8_t>(quantize1(v * Elem<W>::load(w + c) * r, s));
        if (a.h_out != nullptr) static_cast<T *>(a.h_out)[row * a.ldh + c] = Elem<T>::from(v);
    }
}

template <typename T, typename W, int E>
int launch_norm(const lcml_rmsnorm_desc *d, const NormArgs &a, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(d->rows));
    const int64_t nv = d->cols / E;
    // Few rows: one access per thread, the shortest chain from load to store
    // (bf16 64 x 4096: 2.4 us, 2.6 with 256 threads' worth).
    // Many rows: more accesses in flight per thread and smaller reductions
    // (bf16 8000 x 4096: 22.8 us, 33.3 with 1024).
    // At one element per access more warps hide more: 29 -> 18 us for 2000 x 2157 fp16.
    const int want = d->rows <= 2 * sm_count() ? 1024 : (E == 1 ? 512 : 256);
    constexpr int kMost = E == 1 ? 16 : (E * static_cast<int>(sizeof(T)) == 16 ? 4 : 8);
    int vpt = 1;
    while (vpt < kMost && nv > static_cast<int64_t>(vpt) * want) vpt *= 2;
    int64_t threads = ((nv + vpt - 1) / vpt + 31) / 32 * 32;
    if (threads > 1024) {
        return launch_dependent(k_rmsnorm_quantize_long<T, W>, grid, 1024, 0, st, "rmsnorm_quantize_long", a);
    }
    void (*kern)(NormArgs) = nullptr;
    switch (vpt) {
        case 1: kern = k_rmsnorm_quantize<T, W, E, 1>; break;
        case 2: kern = k_rmsnorm_quantize<T, W, E, 2>; break;
        case 4: kern = k_rmsnorm_quantize<T, W, E, 4>; break;
        case 8:
            if constexpr (kMost >= 8) kern = k_rmsnorm_quantize<T, W, E, 8>;
            break;
        case 16:
            if constexpr (kMost >= 16) kern = k_rmsnorm_quantize<T, W, E, 16>;
            break;
    }
    return launch_dependent(kern, grid, static_cast<unsigned>(threads), 0, st, "rmsnorm_quantize", a);
}

template <typename T, typename W>
int dispatch_norm(const lcml_rmsnorm_desc *d, const NormArgs &a, cudaStream_t st) {
    auto fits = [&](int e) {
        const int64_t b = static_cast<int64_t>(e) * static_cast<int64_t>(sizeof(T));
        const uintptr_t al = static_cast<uintptr_t>(b < 16 ? b : 16);
        return d->cols % e == 0 && d->ldx % e == 0 && aligned(d->x, al) && (!d->residual || (d->ldr % e == 0 && aligned(d->residual, al))) &&
               (!d->h_out || (d->ldh % e == 0 && aligned(d->h_out, al))) && aligned(d->weight, e * sizeof(W) < 16 ? e * sizeof(W) : 16) &&
               aligned(d->q, static_cast<uintptr_t>(e));
    };
    if constexpr (sizeof(T) == 2) {
        if (fits(8)) return launch_norm<T, W, 8>(d, a, st);
    }
    if (fits(4)) return launch_norm<T, W, 4>(d, a, st);
    return launch_norm<T, W, 1>(d, a, st);
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" int lcml_rmsnorm_quantize(const lcml_rmsnorm_desc *d, lcml_stream_t stream) {
    LCML_CHECK_ARG(d != nullptr, "lcml_rmsnorm_quantize: null descriptor");
    LCML_CHECK_ARG(d->rows >= 0 && d->cols >= 0, "lcml_rmsnorm_quantize: negative extent");
    LCML_CHECK_ARG(d->x_dtype == LCML_DTYPE_FLOAT || d->x_dtype == LCML_DTYPE_FLOAT16 || d->x_dtype == LCML_DTYPE_BFLOAT16,
                   "lcml_rmsnorm_quantize: x_dtype %d unsupported", d->x_dtype);
    LCML_CHECK_ARG(d->weight_dtype == d->x_dtype || d->weight_dtype == LCML_DTYPE_FLOAT,
                   "lcml_rmsnorm_quantize: weight_dtype %d is neither x's type nor FLOAT", d->weight_dtype);
    LCML_CHECK_ARG(d->eps >= 0.0f, "lcml_rmsnorm_quantize: eps is negative or NaN");
    if (d->rows == 0) return LCML_OK;
    LCML_CHECK_ARG(d->cols > 0, "lcml_rmsnorm_quantize: rows without columns have no norm");
    LCML_CHECK_ARG((d->scale != nullptr) != (d->scale_out != nullptr),
                   "lcml_rmsnorm_quantize: give exactly one of scale and scale_out");
    LCML_CHECK_ARG(d->x && d->weight && d->q, "lcml_rmsnorm_quantize: null pointer");
    LCML_CHECK_ARG(d->rows <= 0x7fffffff && d->cols <= 0x7fffffff, "lcml_rmsnorm_quantize: extent over 2^31 - 1");
    LCML_CHECK_ARG(d->ldx >= d->cols && (!d->residual || d->ldr >= d->cols) && (!d->h_out || d->ldh >= d->cols),
                   "lcml_rmsnorm_quantize: a row stride is less than cols %lld", (long long)d->cols);
    const uintptr_t es = d->x_dtype == LCML_DTYPE_FLOAT ? 4 : 2, ws = d->weight_dtype == LCML_DTYPE_FLOAT ? 4 : 2;
    LCML_CHECK_ARG(aligned(d->x, es) && (!d->residual || aligned(d->residual, es)) && (!d->h_out || aligned(d->h_out, es)) &&
                       aligned(d->weight, ws) && (!d->scale || aligned(d->scale, 4)) && (!d->scale_out || aligned(d->scale_out, 4)),
                   "lcml_rmsnorm_quantize: a pointer is not aligned to its element size");
    const NormArgs a{d->cols, d->ldx, d->ldr, d->ldh, d->x, d->residual, d->h_out, d->weight, d->eps, d->scale, d->scale_out, d->q};
    cudaStream_t st = to_cuda(stream);
    const bool wf = d->weight_dtype == LCML_DTYPE_FLOAT;
    switch (d->x_dtype) {
        case LCML_DTYPE_FLOAT: return dispatch_norm<float, float>(d, a, st);
        case LCML_DTYPE_FLOAT16: return wf ? dispatch_norm<__half, float>(d, a, st) : dispatch_norm<__half, __half>(d, a, st);
        default: return wf ? dispatch_norm<__nv_bfloat16, float>(d, a, st) : dispatch_norm<__nv_bfloat16, __nv_bfloat16>(d, a, st);
    }
}
