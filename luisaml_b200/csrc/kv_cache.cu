// The paged e4m3 key/value cache: quantizing write and read back
// (lcml_kv_cache_write, lcml_kv_cache_read).
//
// Work unit: one block of scale_block positions of one sequence, the span of
// one scale. Sequence b's n tokens touch at most floor(n / block) + 2 blocks,
// so its units start at floor(cu[b] / block) + 2 b (increasing by at least
// that many per sequence): the grid's size follows from host-known totals and
// each CTA finds its sequence by one search in cu_tokens, whatever the
// lengths on the device. A CTA takes one unit and a share of its heads (K and
// V), so the look-ups (sequence, length, page) are paid once per unit.
//
// Bound: the read by HBM (32 x 2000 tokens, 8 heads of 128, to bf16: 61 us, 4.8
// of a copy's 6.5 TB/s; three quarters of its bytes are writes); the write of
// prompts by latency at low occupancy, of loads and of the exact rounding's
// 23 instructions an element (5 prompts of up to 4000 tokens, f16: 38 us, 2.8 TB/s;
// 54 % of the issue slots used, 23 % of the warps active: 64-thread CTAs of 123
// registers); decode steps by the chain of dependent look-ups (cu -> length ->
// page -> codes and scales) of a few L2 latencies, the write's also by the four
// items a CTA takes in turn (one token of 64 sequences, in a graph: write 9.1 us,
// read 5.5).
#include "lcml_decoder.cuh"

namespace lcml {

int check_cache(const lcml_kv_cache *c, const char *what) {
    LCML_CHECK_ARG(c != nullptr, "%s: null cache", what);
    LCML_CHECK_ARG(c->num_pages >= 0 && c->kv_heads > 0 && c->page_size > 0, "%s: bad cache extents", what);
    LCML_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim %d is not 64, 128 or 256", what,
                   c->head_dim);
    LCML_CHECK_ARG(c->scale_block > 0 && c->scale_block % 16 == 0 && c->page_size % c->scale_block == 0,
                   "%s: scale_block %d is not a multiple of 16 that divides page_size %d", what, c->scale_block, c->page_size);
    LCML_CHECK_ARG(static_cast<int64_t>(c->scale_block) * c->head_dim <= 32768, "%s: scale_block * head_dim exceeds 32768", what);
    LCML_CHECK_ARG(c->kv_heads <= 4096 && c->page_size <= 65536 && c->num_pages <= 0x7fffffff / (c->kv_heads * static_cast<int64_t>(c->page_size)),
                   "%s: num_pages * kv_heads * page_size exceeds 2^31 - 1", what);
    if (c->num_pages > 0) {
        LCML_CHECK_ARG(c->k && c->v && c->k_scale && c->v_scale, "%s: null cache pointer", what);
        LCML_CHECK_ARG(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->k_scale, 4) && aligned(c->v_scale, 4),
                       "%s: cache pointers must be 16-byte (codes) and 4-byte (scales) aligned", what);
    }
    return LCML_OK;
}

int check_batch(const lcml_kv_batch *b, const char *what) {
    LCML_CHECK_ARG(b != nullptr, "%s: null batch", what);
    LCML_CHECK_ARG(b->batch >= 0 && b->table_cols >= 0 && b->total_tokens >= 0, "%s: negative extent", what);
    LCML_CHECK_ARG(b->total_tokens <= 0x7fffffff, "%s: too many tokens", what);
    LCML_CHECK_ARG(b->table_stride >= b->table_cols, "%s: table_stride is less than table_cols", what);
    if (b->batch > 0) {
        LCML_CHECK_ARG(b->cu_tokens && b->lengths && (b->block_table || b->table_cols == 0), "%s: null batch pointer", what);
        LCML_CHECK_ARG(aligned(b->cu_tokens, 4) && aligned(b->lengths, 4) && aligned(b->block_table, 4),
                       "%s: a batch pointer is not 4-byte aligned", what);
    }
    return LCML_OK;
}

namespace {

// scale_block * head_dim / 32 threads handle a unit: at most 1024, mostly 256
// or fewer. The write has a second kernel for those, with four times the
// registers: 8 prompts of 2000 tokens, 8 heads of 128 bf16, 38.0 us, 46.3 with
// the large one; one token of 64 sequences 8.4 and 10.7. The read gains nothing
// from one (21.0 and 21.1 us).
constexpr int kSmallUnit = 256, kLargeUnit = 1024;

// One unit as a CTA sees it.
struct Unit {
    int64_t page;      // -1: nothing to do
    int first;         // position of the block's first slot
    int lo, hi;        // the call's tokens in the block, as slots [lo, hi)
    int64_t token;     // packed index of the token in slot lo
    int old;           // slots [0, old) hold earlier tokens
    int slot;          // the block's first slot within its page
};

__device__ __forceinline__ Unit find_unit(const lcml_kv_cache &c, const lcml_kv_batch &b, int64_t u, int *err) {
    Unit r;
    r.page = -1;
    const int blk = c.scale_block;
    const int s = find_sequence(b.cu_tokens, b.batch, u, 1, blk, 2);
    const int t0 = __ldg(b.cu_tokens + s), t1 = min(static_cast<int64_t>(__ldg(b.cu_tokens + s + 1)), b.total_tokens);
    const int start = __ldg(b.lengths + s);
    const int64_t i = u - (t0 / blk + 2 * static_cast<int64_t>(s));  // the sequence's i-th block
    const int64_t first = (static_cast<int64_t>(start) / blk + i) * blk;
    // A sequence without tokens is not looked at further: its table may hold
    // anything, and its last page may be another sequence's to write.
    // i < 0: a unit before the first sequence's, where cu_tokens[0] > 0.
    if (i < 0 || t0 < 0 || t1 <= t0 || start < 0 || first >= static_cast<int64_t>(start) + (t1 - t0)) {
        if (t1 > t0 && start < 0 && threadIdx.x == 0) record_device_error(err, kDevBadBatch);
        return r;
    }
    r.first = static_cast<int>(first);
    r.lo = max(0, start - r.first);
    r.hi = static_cast<int>(min(static_cast<int64_t>(blk), start + static_cast<int64_t>(t1 - t0) - first));
    r.old = r.lo;
    r.token = t0 + (first + r.lo - start);
    const int64_t col = first / c.page_size;
    r.slot = static_cast<int>(first % c.page_size);
    const int64_t page = col < b.table_cols ? __ldg(b.block_table + s * b.table_stride + col) : -1;
    if (page < 0 || page >= c.num_pages) {
        if (threadIdx.x == 0) record_device_error(err, kDevBadPage);
        return r;
    }
    r.page = page;
    return r;
}

struct WriteArgs {
    lcml_kv_cache c;
    lcml_kv_batch b;
    const void *x[2];
    int64_t token_stride[2], head_stride[2];
    int *err;
};

constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100

// RN(v / s) of two values from r = RN(1 / s): Newton steps on the quotient with
// exact fma remainders. By Markstein's theorem (1990) the second one rounds
// correctly, the first having come within an ulp; s within 2^+-60 keeps the
// remainders of every quotient that matters clear of underflow.
__device__ __forceinline__ void divide2(float &q0, float &q1, float v0, float v1, float s, float r) {
    float e0, e1;
    mul2(q0, q1, v0, v1, r, r);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        fma2(e0, e1, q0, q1, -s, -s, v0, v1);
        fma2(q0, q1, e0, e1, r, r, q0, q1);
    }
}

// Bytes 0x7f, 0xff (NaN) and 0x80 of a word of codes, in bit 7 of each byte.
__device__ __forceinline__ uint32_t special_bytes(uint32_t w) {
    const uint32_t m = w & 0x7f7f7f7fu;
    return ((m + 0x01010101u) | (~(m + 0x7f7f7f7fu) & w)) & 0x80808080u;
}

// QuantizeLinear of 8 values, bit-identical to quantize1(). As
// quantize_block_fast(): where the codes of v * r_lo and v * r_hi agree they
// are the code of RN(v / s). 16-bit inputs meet a rounding boundary often (448
// = 7 * 64: for a bf16 maximum with an even significand one significand in 128
// divides to the midpoint 21/16), so a block with a disagreement is divided
// correctly in place, and only one with NaN or 0x80 codes, or an unusual
// scale, takes the scalar divide and the integer encoder.
__device__ __forceinline__ void quantize8(const float *v, float s, float r, bool s_ok, uint32_t *w) {
    const float r_lo = r * 0.99999952316284180f;  // 1 - 2^-21
    const float r_hi = r * 1.00000047683715820f;  // 1 + 2^-21
    uint32_t other[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            fma2(lo[k], lo[k + 1], v[4 * j + k], v[4 * j + k + 1], r_lo, r_lo, 0.0f, 0.0f);
            fma2(hi[k], hi[k + 1], v[4 * j + k], v[4 * j + k + 1], r_hi, r_hi, 0.0f, 0.0f);
        }
        w[j] = cvt_e4m3x2(lo[0], lo[1]) | (cvt_e4m3x2(lo[2], lo[3]) << 16);
        other[j] = cvt_e4m3x2(hi[0], hi[1]) | (cvt_e4m3x2(hi[2], hi[3]) << 16);
    }
    if (((w[0] ^ other[0]) | (w[1] ^ other[1])) != 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float q[4];
            divide2(q[0], q[1], v[4 * j], v[4 * j + 1], s, r);
            divide2(q[2], q[3], v[4 * j + 2], v[4 * j + 3], s, r);
            w[j] = cvt_e4m3x2(q[0], q[1]) | (cvt_e4m3x2(q[2], q[3]) << 16);
        }
    }
    if ((special_bytes(w[0]) | special_bytes(w[1])) != 0 || !s_ok) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            w[j] = quantize1(v[4 * j], s) | (quantize1(v[4 * j + 1], s) << 8) | (quantize1(v[4 * j + 2], s) << 16) | (quantize1(v[4 * j + 3], s) << 24);
    }
}

// The unit's new values stay in registers (kVpt vectors of 8 per thread)
// between the maximum and the encoding, so they are read once; the next item's
// are on their way meanwhile.
constexpr int kVpt = 4;

template <typename T, bool VEC>
struct Row8 {
    T e[8];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC && sizeof(T) == 2) {
            *reinterpret_cast<uint4 *>(e) = __ldcs(reinterpret_cast<const uint4 *>(p));
        } else if constexpr (VEC) {
            reinterpret_cast<uint4 *>(e)[0] = __ldcs(reinterpret_cast<const uint4 *>(p));
            reinterpret_cast<uint4 *>(e)[1] = __ldcs(reinterpret_cast<const uint4 *>(p) + 1);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
};

template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) k_kv_cache_write(WriteArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    __shared__ uint32_t red[2][32];
    const Unit un = find_unit(a.c, a.b, blockIdx.x, a.err);
    if (un.page < 0) return;
    const int hk = a.c.kv_heads, d = a.c.head_dim, blk = a.c.scale_block, per_row = d >> 3;
    const int shift = d == 64 ? 3 : (d == 128 ? 4 : 5);  // per_row = 1 << shift
    const int nv = (un.hi - un.lo) * per_row;            // vectors of new values
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int64_t base0 = un.page * hk * a.c.page_size + un.slot;
    alignas(16) Row8<T, VEC> raw[kVpt];
    float s_old;
    auto fetch = [&](int item) {
        const int kv = item >= hk ? 1 : 0, head = item - kv * hk;
        const T *x = static_cast<const T *>(a.x[kv]) + un.token * a.token_stride[kv] + head * a.head_stride[kv];
#pragma unroll
        for (int j = 0; j < kVpt; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < nv) raw[j].load(x + (i >> shift) * a.token_stride[kv] + ((i & (per_row - 1)) << 3));
        }
        s_old = un.old > 0 ? (kv ? a.c.v_scale : a.c.k_scale)[(base0 + static_cast<int64_t>(head) * a.c.page_size) / blk] : 0.0f;
    };
    int item = blockIdx.y;
    fetch(item);
    for (int turn = 0; item < 2 * hk; item += gridDim.y, turn ^= 1) {
        const int kv = item >= hk ? 1 : 0, head = item - kv * hk;
        const int64_t base = base0 + static_cast<int64_t>(head) * a.c.page_size;
        uint8_t *codes = (kv ? a.c.v : a.c.k) + base * d;
        float *scale = (kv ? a.c.v_scale : a.c.k_scale) + base / blk;
        float v[kVpt][8];
        const float had = s_old;
        float mx = 0.0f;  // fmaxf ignores NaN
#pragma unroll
        for (int j = 0; j < kVpt; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < nv) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    v[j][e] = Elem<T>::load(raw[j].e + e);
                    v[j][e + 1] = Elem<T>::load(raw[j].e + e + 1);
                    mx = fmaxf(fmaxf(mx, fabsf(v[j][e])), fabsf(v[j][e + 1]));
                }
            }
        }
        if (mx == INFINITY) {  // an infinity does not count
            mx = 0.0f;
#pragma unroll
            for (int j = 0; j < kVpt; ++j)
                if (static_cast<int>(threadIdx.x + j * blockDim.x) < nv) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (fabsf(v[j][e]) < INFINITY) mx = fmaxf(mx, fabsf(v[j][e]));
                }
        }
        if (item + gridDim.y < 2 * hk) fetch(item + gridDim.y);
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));  // floats >= 0 order like their bits
        if (nw > 1) {  // two buffers in turn: one barrier per item
            if (l == 0) red[turn][w] = bits;
            __syncthreads();
            bits = __reduce_max_sync(0xffffffffu, l < nw ? red[turn][l] : 0u);
        }
        const float amax = __uint_as_float(bits);
        float s = amax > 0.0f ? fmaxf(__fdiv_rn(amax, 448.0f), kMinScale) : 0.0f;
        const bool grew = un.old > 0 && s > had;
        s = fmaxf(s, had);
        const float div = s > 0.0f ? s : 1.0f;
        const float r = __frcp_rn(div);
        const bool ok = div >= 8.673617379884035e-19f && div <= 1.152921504606847e18f;  // 2^+-60: divide2()
#pragma unroll
        for (int j = 0; j < kVpt; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < nv) {
                uint32_t q[2];
                quantize8(v[j], div, r, ok, q);
                *reinterpret_cast<uint2 *>(codes + (un.lo + (i >> shift)) * d + ((i & (per_row - 1)) << 3)) = make_uint2(q[0], q[1]);
            }
        }
        if (grew) {  // the earlier codes move to the new scale
            for (int i = threadIdx.x; i < un.old * per_row; i += blockDim.x) {
                uint2 *p = reinterpret_cast<uint2 *>(codes) + i;
                const uint2 c = *p;
                float f[8];
                e4m3x2_decode(c.x & 0xffffu, f[0], f[1]);
                e4m3x2_decode(c.x >> 16, f[2], f[3]);
                e4m3x2_decode(c.y & 0xffffu, f[4], f[5]);
                e4m3x2_decode(c.y >> 16, f[6], f[7]);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= had;
                uint32_t q[2];
                quantize8(f, div, r, ok, q);
                *p = make_uint2(q[0], q[1]);
            }
        }
        // every thread has read the old scale before the barrier above (nw > 1) or in lockstep (one warp)
        if (nw == 1) __syncwarp();
        if (threadIdx.x == 0) *scale = s;
    }
}

struct ReadArgs {
    lcml_kv_cache c;
    lcml_kv_batch b;
    void *y[2];
    int *err;
};

template <typename T>
__global__ void __launch_bounds__(kLargeUnit) k_kv_cache_read(ReadArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const Unit un = find_unit(a.c, a.b, blockIdx.x, a.err);
    if (un.page < 0) return;
    const int hk = a.c.kv_heads, d = a.c.head_dim, blk = a.c.scale_block;
    const int shift = d == 64 ? 3 : (d == 128 ? 4 : 5);
    const int nv = (un.hi - un.lo) << shift;
    // a thread's codes of one item: 16 at a time, twice (blockDim.x * 32 codes cover a unit)
    constexpr int kPer = kVpt / 2;
    const int shift16 = shift - 1, per16 = 1 << shift16, n16 = nv >> 1;
    const int64_t base0 = un.page * hk * a.c.page_size + un.slot;
    uint4 c[kPer];
    float s;
    auto fetch = [&](int item) {
        const int kv = item >= hk ? 1 : 0, head = item - kv * hk;
        const int64_t base = base0 + static_cast<int64_t>(head) * a.c.page_size;
        const uint4 *codes = reinterpret_cast<const uint4 *>((kv ? a.c.v : a.c.k) + (base + un.lo) * d);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < n16) c[j] = __ldg(codes + i);
        }
        s = __ldg((kv ? a.c.v_scale : a.c.k_scale) + base / blk);
    };
    int item = blockIdx.y;
    fetch(item);
    for (; item < 2 * hk; item += gridDim.y) {
        const int kv = item >= hk ? 1 : 0, head = item - kv * hk;
        uint4 now[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) now[j] = c[j];
        const float scale = s;
        if (item + gridDim.y < 2 * hk) fetch(item + gridDim.y);
        if (a.y[kv] == nullptr) continue;
        T *y = static_cast<T *>(a.y[kv]) + (un.token * hk + head) * d;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < n16) {
                const uint32_t cw[4] = {now[j].x, now[j].y, now[j].z, now[j].w};
                float f[16];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    e4m3x2_decode(cw[q] & 0xffffu, f[4 * q], f[4 * q + 1]);
                    e4m3x2_decode(cw[q] >> 16, f[4 * q + 2], f[4 * q + 3]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] *= scale;
                store_vec<T, 16>(y + static_cast<int64_t>(i >> shift16) * hk * d + ((i & (per16 - 1)) << 4), f);
            }
        }
    }
}

unsigned unit_threads(const lcml_kv_cache *c) { return static_cast<unsigned>(c->scale_block * c->head_dim / (8 * kVpt)); }

// grid.x: units; grid.y: how many CTAs share a unit's 2 * kv_heads items. Where
// one wave of CTAs has room for several per unit, as many as fit (a second
// wave would wait for the first one's look-ups: 15 -> 9 us for 64 tokens of 64
// sequences); for more units two waves, so that the last one is a small part.
dim3 unit_grid(const lcml_kv_cache *c, const lcml_kv_batch *b) {
    const int64_t units = b->total_tokens / c->scale_block + 2 * static_cast<int64_t>(b->batch);
    const int64_t per_sm = 2048 / unit_threads(c) < 32 ? 2048 / unit_threads(c) : 32;
    const int64_t wave = per_sm * sm_count() / 2;  // the registers let about half of the threads in
    int64_t y = wave / units >= 4 ? wave / units : (4 * wave + units - 1) / units;
    if (y > 2 * c->kv_heads) y = 2 * c->kv_heads;
    return dim3(static_cast<unsigned>(units), static_cast<unsigned>(y < 1 ? 1 : y));
}

template <typename T>
int launch_write(const lcml_kv_cache *c, const lcml_kv_batch *b, const WriteArgs &a, bool vec, cudaStream_t st) {
    auto kern = unit_threads(c) <= kSmallUnit ? (vec ? k_kv_cache_write<T, true, kSmallUnit> : k_kv_cache_write<T, false, kSmallUnit>)
                                              : (vec ? k_kv_cache_write<T, true, kLargeUnit> : k_kv_cache_write<T, false, kLargeUnit>);
    return launch_dependent(kern, unit_grid(c, b), unit_threads(c), 0, st, "kv_cache_write", a);
}

template <typename T>
int launch_read(const lcml_kv_cache *c, const lcml_kv_batch *b, const ReadArgs &a, cudaStream_t st) {
    auto kern = k_kv_cache_read<T>;
    return launch_dependent(kern, unit_grid(c, b), unit_threads(c), 0, st, "kv_cache_read", a);
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" {

int lcml_kv_cache_write(const lcml_kv_cache *cache, const lcml_kv_batch *batch, const void *k, int64_t k_token_stride,
                        int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                        lcml_stream_t stream) {
    int rc = check_cache(cache, "lcml_kv_cache_write");
    if (rc == LCML_OK) rc = check_batch(batch, "lcml_kv_cache_write");
    if (rc != LCML_OK) return rc;
    LCML_CHECK_ARG(dtype == LCML_DTYPE_FLOAT || dtype == LCML_DTYPE_FLOAT16 || dtype == LCML_DTYPE_BFLOAT16,
                   "lcml_kv_cache_write: dtype %d unsupported", dtype);
    if (batch->batch == 0 || batch->total_tokens == 0) return LCML_OK;
    LCML_CHECK_ARG(k && v, "lcml_kv_cache_write: null pointer");
    LCML_CHECK_ARG(k_token_stride >= 0 && k_head_stride >= 0 && v_token_stride >= 0 && v_head_stride >= 0,
                   "lcml_kv_cache_write: negative stride");
    const int64_t es = dtype == LCML_DTYPE_FLOAT ? 4 : 2;
    LCML_CHECK_ARG(aligned(k, es) && aligned(v, es), "lcml_kv_cache_write: k or v is not aligned to its element size");
    const int64_t e16 = 16 / es;
    const bool vec = aligned(k, 16) && aligned(v, 16) && k_token_stride % e16 == 0 && k_head_stride % e16 == 0 &&
                     v_token_stride % e16 == 0 && v_head_stride % e16 == 0;
    const WriteArgs a{*cache, *batch, {k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, device_error_word()};
    cudaStream_t st = to_cuda(stream);
    if (dtype == LCML_DTYPE_FLOAT) return launch_write<float>(cache, batch, a, vec, st);
    if (dtype == LCML_DTYPE_FLOAT16) return launch_write<__half>(cache, batch, a, vec, st);
    return launch_write<__nv_bfloat16>(cache, batch, a, vec, st);
}

int lcml_kv_cache_read(const lcml_kv_cache *cache, const lcml_kv_batch *batch, void *k, void *v, int dtype,
                       lcml_stream_t stream) {
    int rc = check_cache(cache, "lcml_kv_cache_read");
    if (rc == LCML_OK) rc = check_batch(batch, "lcml_kv_cache_read");
    if (rc != LCML_OK) return rc;
    LCML_CHECK_ARG(dtype == LCML_DTYPE_FLOAT || dtype == LCML_DTYPE_FLOAT16 || dtype == LCML_DTYPE_BFLOAT16,
                   "lcml_kv_cache_read: dtype %d unsupported", dtype);
    if (batch->batch == 0 || batch->total_tokens == 0) return LCML_OK;
    LCML_CHECK_ARG(k || v, "lcml_kv_cache_read: null pointers");
    LCML_CHECK_ARG(aligned(k, 16) && aligned(v, 16), "lcml_kv_cache_read: k and v must be 16-byte aligned");
    const ReadArgs a{*cache, *batch, {k, v}, device_error_word()};
    cudaStream_t st = to_cuda(stream);
    if (dtype == LCML_DTYPE_FLOAT) return launch_read<float>(cache, batch, a, st);
    if (dtype == LCML_DTYPE_FLOAT16) return launch_read<__half>(cache, batch, a, st);
    return launch_read<__nv_bfloat16>(cache, batch, a, st);
}

}// extern "C"
