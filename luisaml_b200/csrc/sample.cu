// The next token of every row of logits (lcml_sample): temperature, top-k, top-p,
// min-p, then the draw from a given uniform number.
//
// One cluster of CTAs per row; the row is read once and stays in the cluster's
// shared memory (rows too long for that are read again from L2). What top-k,
// top-p and min-p keep is a prefix of the tokens by falling logit, so each comes
// down to its last token, the cut (x, index). No sort of the row finds it:
//   top-k: the k-th largest of the threads' own largest logits (a histogram of one
//      value a thread) bounds the cut from below with few tokens above it. They
//      go into a list, and top-p is taken from it right away.
//   top-p: the pass that sums all weights also bins them, 64 bins to a factor of two,
//      in 32-bit units of the bin's own weight: that says to 1e-4 of the sum in
//      which bin the kept mass passes its target. A second pass sums the weights
//      before that bin exactly and lists its tokens.
// The list is in every CTA, so each finds the cut for itself. Where it is too short,
// or the cut lies elsewhere after all, cut_slow() narrows the range step by step.
// The draw needs no order either: weights of the kept tokens summed by rising
// index, per warp, then the CTA that holds uniform * sum goes over that warp's tokens
// once more. Up to 256 kept tokens are all in the list and drawn from there.
//
// Weights and sums are fp64, in an order that the sizes, the number of rows and the row's
// alignment fix (of the list, whose order atomics make, as 64-bit integers or sorted): a token lies within an fp32 rounding
// of its neighbours' range once in some thousand rows, and the result would go by
// the order of the sum. Where few tokens count they are packed 32 to a warp before
// they are weighed (Queue).
//
// Bound: the phases of a row, one after the other, and their instructions (128 rows of 128001
// with top_p: 63 % of the issue slots, 18 % of the fp64 pipe). Of a row of 128001 fp32 logits in
// one CTA, 128 of them beside each other, 12,000 clocks go to the load, 45,000 to the
// weights (13 fp64 instructions a token and 30 others), 14,000 to their bins, 25,000 to
// the pass for the cut at top_p 0.9 (more the more tokens that keeps) and 15,000 to the
// rest: 77 us, 39 without top_p, 23 with top_k 50 (floor 10). Small calls are a chain of some
// ten barriers and fp64 sums: 14 us for a row of 2000 with top_p, 11 for one of 32000 with top_k.
#include <type_traits>

#include "lcml_decoder.cuh"

#include "../../include/lcml_decode_step.h"

namespace lcml {
namespace {

constexpr int kMaxCluster = 4;  // CTAs a row
constexpr int kBins = 2048;
constexpr int kList = 1024;  // tokens whose order is found in one CTA
constexpr int kPairs = 256;  // of which so many by comparing each with each
constexpr uint32_t kOneBits = 0x3ff00000u;  // the upper word of 1.0
constexpr int kBinShift = 14;  // a bin of the weights' histogram: their upper words but for these bits
constexpr unsigned kAll = 0xffffffffu;
constexpr float kLowest = -3.402823466385288598e38f;  // the least finite float, which masks use

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int vocab, slice;  // tokens, and how many of them a CTA takes
    int ctas;          // per row
    const float *uniform, *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    int32_t *tokens;
    float *logprob;
};

template <int NT>
struct alignas(16) Shared {
    static constexpr int kWarps = NT / 32;
    unsigned long long slot[2][kMaxCluster * kWarps][2];  // what the row's warps tell each other, two turns
    float queue_x[kWarps][32 * 5];
    int queue_index[kWarps][32 * 5];
    unsigned long long list[kList];
    uint32_t bins[kBins];
    float scan_f[kWarps];
    uint32_t scan_u[kWarps];
    double scan[kWarps];
    unsigned long long part[kPairs], total;
    int first, last, filled;      // found bins or places of the list
    uint32_t under;               // sum before the first one
    unsigned long long verdict;   // from the CTA that finds it
    uint32_t listed[2];           // in rank 0: tokens in the list, of two passes
};

template <int NT>
constexpr int kShared = static_cast<int>(sizeof(Shared<NT>));
template <int NT>
constexpr int kStageMost = 227 * 1024 - kShared<NT>;  // of a row, in the shared memory of a CTA

// Order-preserving bits of a float (no NaN).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A token in the order: falling logit (-0 is 0), equal ones by rising index.
__device__ __forceinline__ unsigned long long entry_of(float x, int index) {
    return static_cast<unsigned long long>(key_of(x + 0.0f)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

struct Weight {
    double top, per;  // largest logit, log2(e) / temperature
    float least;      // logits below it weigh nothing
    // 2^t, t = (x - top) per: t's nearest whole number by addition of 1.5 2^52, 2^f of the rest
    // on [-1/2, 1/2] as 1 + f p(f), p fitted at Chebyshev points with 2^f's relative
    // error as the weight (8.2e-13), so the largest logit has exactly 1.
    __device__ __forceinline__ double operator()(float x) const {
        const double d = static_cast<double>(x) - top, s = fma(d, per, 6755399441055744.0);
        const double f = fma(d, per, 6755399441055744.0 - s);
        double p = 1.3178918944060163e-06;
        p = fma(p, f, 1.5309155627301653e-05);
        p = fma(p, f, 0.00015403825519790757);
        p = fma(p, f, 0.0013333454862616348);
        p = fma(p, f, 0.009618128616057417);
        p = fma(p, f, 0.055504109352640572);
        p = fma(p, f, 0.24022650698110781);
        p = fma(p, f, 0.69314718054821356);
        p = fma(p, f, 1.0);
        return counts(x) ? __hiloint2double(__double2hiint(p) + (__double2loint(s) << 20), __double2loint(p)) : 0.0;
    }
    __device__ __forceinline__ bool counts(float x) const { return x >= least; }  // not NaN, not -infinity
};

__device__ __forceinline__ void st_cluster(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint2 ld_cluster_u2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t add_cluster(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ double warp_upto(double v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(kAll, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// Packs few of a warp's many tokens, so that 32 of them are worked on together.
struct Queue {
    float *x;        // 32 * kAtOnce + 32 of each
    int *index;
    int lane;
    int held = 0;
    static constexpr int kAtOnce = 4;

    // Adds the marked ones of kAtOnce tokens per lane; calls f(logit, index, whether the lane has one) for 32 at a time.
    template <typename F>
    __device__ __forceinline__ void push(const float *v, int i, uint32_t marked, F f) {
        uint32_t m[kAtOnce];
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) m[e] = __ballot_sync(kAll, marked >> e & 1u);
        if ((m[0] | m[1] | m[2] | m[3]) == 0) return;
        static_assert(kAtOnce == 4, "four masks");
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
            const int at = held + __popc(m[e] & ((1u << lane) - 1));
            if (marked >> e & 1u) {
                x[at] = v[e];
                index[at] = i + e;
            }
            held += __popc(m[e]);
        }
        if (held < 32) return;
        __syncwarp();
        int from = 0;
        for (; held - from >= 32; from += 32) f(x[from + lane], index[from + lane], true);
        const bool rest = from + lane < held;
        const float y = rest ? x[from + lane] : 0.0f;
        const int j = rest ? index[from + lane] : 0;
        __syncwarp();
        if (rest) {
            x[lane] = y;
            index[lane] = j;
        }
        held -= from;
    }
    template <typename F>
    __device__ __forceinline__ void flush(F f) {
        if (held == 0) return;
        __syncwarp();
        f(x[lane], index[lane], lane < held);
        __syncwarp();
        held = 0;
    }
};

// What a row's CTA works with.
template <typename T, bool STAGED, int NT>
struct Row {
    static constexpr int kWarps = NT / 32, kPer = kBins / NT;
    static constexpr int E = 16 / static_cast<int>(sizeof(T));  // tokens a lane takes at once
    static constexpr int kStep = 32 * E;
    static constexpr int kAhead = E == 4 ? 4 : 2;
    using Told = const unsigned long long (*)[2];

    const SampleArgs &a;
    Shared<NT> &sh;
    T *stage;        // the CTA's slice
    const T *x;      // the row
    int off;         // tokens by which the row begins after a 16-byte boundary
    int rank, lane, warp;
    int turn = 0;
    Weight weight;
    // bins of equal width, or of keys: see set_bins()
    float hi, scale;
    uint32_t k_hi;
    int shift;
    bool linear;

    // Tokens are counted from the boundary before the row, so that every lane's
    // E are one 16-byte access, but for the row's ends.
    __device__ __forceinline__ int64_t warp_first() const {
        return static_cast<int64_t>(rank) * a.slice + warp * (a.slice / kWarps);
    }
    __device__ __forceinline__ int steps() const {
        const int64_t left = static_cast<int64_t>(a.vocab) + off - warp_first();
        const int most = a.slice / kWarps / kStep;
        return left <= 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(most), (left + kStep - 1) / kStep));
    }
    __device__ __forceinline__ int index_of(int s) const {  // of the lane's first token in step s; below 0 or past the row: none
        return static_cast<int>(warp_first() + static_cast<int64_t>(s) * kStep + lane * E - off);
    }
    __device__ __forceinline__ bool own_warp(int index) const {  // whether the token is among this warp's
        const int64_t at = static_cast<int64_t>(index) + off - warp_first();
        return at >= 0 && at < a.slice / kWarps;
    }
    __device__ __forceinline__ void fetch(int s, T (&t)[E]) const {
        const int i = index_of(s);
        if (i >= 0 && i + E <= a.vocab) {
            *reinterpret_cast<uint4 *>(t) = __ldg(reinterpret_cast<const uint4 *>(x + i));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] = i + e >= 0 && i + e < a.vocab ? x[i + e] : Elem<T>::from(-INFINITY);
        }
    }
    __device__ __forceinline__ T *staged(int s) const { return stage + warp * (a.slice / kWarps) + s * kStep + lane * E; }
    __device__ __forceinline__ void load(int s, float (&v)[E]) const {
        alignas(16) T t[E];
        if constexpr (STAGED) *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(staged(s));
        else fetch(s, t);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = Elem<T>::load(t + e);
    }
    // Calls f(logits, index of the first) for each of the warp's steps, kAhead of which are loaded at once.
    template <typename F>
    __device__ __forceinline__ void sweep(F f) const {
        const int n = steps(), i0 = index_of(0);
        // steps whose lanes all lie within the row
        const int from = STAGED || i0 - lane * E >= 0 ? 0 : 1, to = STAGED ? n : min(n, max(from, (a.vocab - (i0 - lane * E)) / kStep));
        const T *p = STAGED ? staged(0) : x + i0;
        auto one = [&](const T(&t)[E], int i) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = Elem<T>::load(t + e);
            f(v, i);
        };
        int s = from;
#pragma unroll 1
        for (; s + kAhead <= to; s += kAhead) {
            alignas(16) T t[kAhead][E];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const uint4 *q = reinterpret_cast<const uint4 *>(p + (s + j) * kStep);
                *reinterpret_cast<uint4 *>(t[j]) = STAGED ? *q : __ldg(q);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) one(t[j], i0 + (s + j) * kStep);
        }
#pragma unroll 1
        for (const int rest = n - s + from, first = s; s - first < rest; ++s) {  // those left over, and a first one that begins before the row
            const int u = s < n ? s : 0;
            alignas(16) T t[E];
            if constexpr (STAGED) *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(staged(u));
            else fetch(u, t);
            one(t, i0 + u * kStep);
        }
    }
    // Calls f(logit, index, whether the lane has one) with the tokens that `in` marks, packed.
    template <typename M, typename F>
    __device__ __forceinline__ void pick(M in, F f) const {
        Queue q{sh.queue_x[warp], sh.queue_index[warp], lane};
        sweep([&](const float(&v)[E], int i) {
#pragma unroll
            for (int h = 0; h < E; h += Queue::kAtOnce) {
                uint32_t marked = 0;
#pragma unroll
                for (int e = 0; e < Queue::kAtOnce; ++e) marked |= in(v[h + e], i + h + e) ? 1u << e : 0u;
                q.push(v + h, i + h, marked, f);
            }
        });
        q.flush(f);
    }

    // Exchange of two values per warp (the same in its lanes): every thread may read
    // them all, in the order of the tokens. The barrier also makes what was stored
    // into other CTAs before it visible there.
    __device__ __forceinline__ Told tell(unsigned long long v0, unsigned long long v1) {
        say(v0, v1);
        return hear();
    }
    __device__ __forceinline__ void say(unsigned long long v0, unsigned long long v1) {
        if (lane < a.ctas) {
            const uint32_t to = mapa_shared(smem_u32(&sh.slot[turn][rank * kWarps + warp][0]), lane);
            st_cluster(to, v0);
            st_cluster(to + 8, v1);
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    }
    __device__ __forceinline__ Told hear() {
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        const Told got = sh.slot[turn];
        turn ^= 1;
        return got;
    }
    // Over the row's warps: the largest and the sum of the lower or upper halves of what they told, and the sum as fp64.
    __device__ __forceinline__ uint32_t largest(Told got, int which, int half) const {
        uint32_t v = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster * kWarps / 32; ++r)
            if (r * 32 + lane < a.ctas * kWarps) v = max(v, static_cast<uint32_t>(got[r * 32 + lane][which] >> (32 * half)));
        return __reduce_max_sync(kAll, v);
    }
    __device__ __forceinline__ uint32_t count_of(Told got) const {
        uint32_t v = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster * kWarps / 32; ++r)
            if (r * 32 + lane < a.ctas * kWarps) v += static_cast<uint32_t>(got[r * 32 + lane][1]);
        return __reduce_add_sync(kAll, v);
    }
    __device__ __forceinline__ double sum_of(Told got) const {
        double v = 0.0;
#pragma unroll
        for (int r = 0; r < kMaxCluster * kWarps / 32; ++r)
            if (r * 32 + lane < a.ctas * kWarps) v += __longlong_as_double(got[r * 32 + lane][0]);
        return warp_sum(v);
    }

    // Sum of the weights of the warp's tokens, all of them, or the few that `keep` takes.
    __device__ __forceinline__ double mass_of_all() const {
        double sum = 0.0;
        sweep([&](const float(&v)[E], int) {
            double w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = weight(v[e]);
#pragma unroll
            for (int e = 0; e < E; ++e) sum += w[e];
        });
        return warp_sum(sum);
    }
    template <typename F>
    __device__ __forceinline__ double mass_of(F keep) const {
        double sum = 0.0;
        pick(keep, [&](float y, int, bool is) {
            const double w = weight(y);
            sum += is ? w : 0.0;
        });
        return warp_sum(sum);
    }

    // Bins of equal width, or by the bits of the logit where these are few: then a
    // bin is one value. lo and hi lie in different bins, so every turn narrows.
    __device__ __forceinline__ void set_bins(float lo, float to) {
        hi = to + 0.0f;
        k_hi = key_of(hi);
        const uint32_t range = k_hi - key_of(lo + 0.0f);
        linear = range >= kBins && hi * 0.5f - lo * 0.5f > 1e-30f;
        scale = linear ? kBins / (hi * 0.5f - lo * 0.5f) : 0.0f;
        shift = max(0, 32 - __clz(range) - 11);
        static_assert(kBins == 1 << 11, "eleven bits a turn");
    }
    __device__ __forceinline__ int bin(float v) const {
        return linear ? static_cast<int>(fminf((hi * 0.5f - v * 0.5f) * scale, kBins - 1.0f)) : static_cast<int>((k_hi - key_of(v + 0.0f)) >> shift);
    }
    // A value that no logit of bins 0 .. b is below; low: the least logit that was binned.
    __device__ __forceinline__ float edge_below(int b, float low) const {
        if (!linear) return b >= kBins - 1 ? low : value_of(max(key_of(low), k_hi - ((static_cast<uint32_t>(b) + 1) << shift) + 1));
        // the difference and the product are rounded by 2^-24 each
        return fmaxf(low, static_cast<float>(hi - 2.0 * (b + 1) / scale * (1.0 + 1e-6) - 1e-6 * fabs(static_cast<double>(hi))));
    }
    // About the logit whose weight is the upper edge of bin b of the weights.
    __device__ __forceinline__ float edge_above(int b) const {
        return static_cast<float>(weight.top) + log2f(__hiloint2double((kOneBits >> kBinShift) - b + 1 << kBinShift, 0)) / static_cast<float>(weight.per);
    }
    __device__ __forceinline__ void clear_bins() {
        for (int i = threadIdx.x; i < kBins / 2; i += NT) reinterpret_cast<uint2 *>(sh.bins)[i] = make_uint2(0, 0);
        if (threadIdx.x == 0) {
            sh.first = sh.last = kBins;
            sh.filled = 0;
        }
        __syncthreads();
    }
    // The counts of kPer bins a thread, from all CTAs (after a barrier of the cluster).
    template <typename U>
    __device__ __forceinline__ void all_bins(U (&c)[kPer]) {
        const uint32_t at = smem_u32(&sh.bins[kPer * threadIdx.x]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) c[j] = 0;
#pragma unroll
        for (int j = 0; j < kPer; j += 2) {
            uint2 u[kMaxCluster];
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r)
                if (r < a.ctas) u[r] = ld_cluster_u2(mapa_shared(at + 4 * j, r));
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r)
                if (r < a.ctas) {
                    c[j] += u[r].x;
                    c[j + 1] += u[r].y;
                }
        }
    }
    // The first bin up to which the row's bins hold `want` or more (kBins: none), sh.under: how
    // many the bins before it hold, sh.filled: the last bin that holds anything.
    __device__ __forceinline__ int find_bin(uint32_t want) {
        uint32_t c[kPer], mine = 0;
        all_bins(c);
        const int b = kPer * threadIdx.x;
        int filled = -1;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            mine += c[j];
            filled = c[j] != 0 ? b + j : filled;
        }
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(kAll, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) sh.scan_u[warp] = upto;
        __syncthreads();
        upto += __reduce_add_sync(kAll, lane < warp ? sh.scan_u[lane] : 0u);
        if (filled >= 0) atomicMax(&sh.filled, filled);
        uint32_t under = upto - mine;
        if (under < want && upto >= want) {  // in one thread
            int j = 0;
#pragma unroll
            for (int q = 0; q < kPer - 1; ++q)
                if (j == q && under + c[q] < want) {
                    under += c[q];
                    ++j;
                }
            sh.first = b + j;
            sh.under = under;
        }
        __syncthreads();
        return sh.first;
    }
    // All lanes: those with `in` put their token into the list of every CTA. which: the pass.
    __device__ __forceinline__ void list(float v, int i, bool in, int which) {
        const uint32_t m = __ballot_sync(kAll, in);
        if (m == 0) return;
        const bool one = a.ctas == 1;  // CTA: without the way round by the cluster
        uint32_t at = 0;
        if (lane == 0) at = one ? atomicAdd(&sh.listed[which], __popc(m)) : add_cluster(mapa_shared(smem_u32(&sh.listed[which]), 0), __popc(m));
        at = __shfl_sync(kAll, at, 0) + __popc(m & ((1u << lane) - 1));
        if (in && at < kList) {
            if (one) {
                sh.list[at] = entry_of(v, i);
            } else {
                for (int r = 0; r < a.ctas; ++r) st_cluster(mapa_shared(smem_u32(&sh.list[0]), r) + at * 8, entry_of(v, i));
            }
        }
    }

    // A listed token's weight in units of 2^-52, at least one of what weighs anything.
    __device__ __forceinline__ unsigned long long units_of(unsigned long long entry) const {
        const double w = weight(value_of(static_cast<uint32_t>(entry >> 32)));
        return max(static_cast<unsigned long long>(w * 0x1p52), w > 0.0 ? 1ull : 0ull);
    }
    // The cut of the first `want` (kCount) of the n listed tokens and, top_p below 1, of the fewest first ones
    // of those whose weights sum to top_p of theirs; or (not kCount) of the fewest first ones whose
    // weights and `above` reach `target`. 0: none does, though there are n.
    template <bool kCount>
    __device__ __forceinline__ unsigned long long cut_of_list(uint32_t n, uint32_t want, double above, double target, double top_p) {
        if (n == 0) return 0;
        if (n <= kPairs) {
            // Each with each, four threads a token: its rank and the weights before it, in units
            // of 2^-52 (exact sums, whatever the list's order).
            const int q = threadIdx.x & 3;
            const uint32_t stays = min(want, n);
            for (uint32_t i = threadIdx.x; i < n; i += NT) sh.part[i] = units_of(sh.list[i]);
            if (threadIdx.x == 0) sh.verdict = 0;
            __syncthreads();
            auto place = [&](uint32_t t, unsigned long long &before) {
                const unsigned long long mine = t < n ? sh.list[t] : ~0ull;
                uint32_t rank_of = 0;
                before = 0;
                for (uint32_t j = q; j < n; j += 4) {
                    const bool ahead = sh.list[j] > mine;
                    before += ahead ? sh.part[j] : 0;
                    rank_of += ahead;
                }
#pragma unroll
                for (int o = 1; o < 4; o *= 2) {
                    before += __shfl_xor_sync(kAll, before, o);
                    rank_of += __shfl_xor_sync(kAll, rank_of, o);
                }
                return rank_of;
            };
            constexpr int kTurns = 4 * kPairs / NT;
            unsigned long long before[kTurns];
            uint32_t rank_of[kTurns];
#pragma unroll
            for (int u = 0; u < kTurns; ++u) {
                const uint32_t t = threadIdx.x / 4 + u * (NT / 4);
                if (u * (NT / 4) < static_cast<int>(n)) rank_of[u] = place(t, before[u]);
                if (kCount && t < n && q == 0 && rank_of[u] == stays - 1) sh.total = before[u] + sh.part[t];  // of all that stay
            }
            if (kCount && top_p < 1.0) {
                __syncthreads();
                target = top_p * static_cast<double>(sh.total);
            }
#pragma unroll
            for (int u = 0; u < kTurns; ++u) {
                const uint32_t t = threadIdx.x / 4 + u * (NT / 4);
                if (t >= n || q != 0) continue;
                const double from = static_cast<double>(before[u]), to = static_cast<double>(before[u] + sh.part[t]);
                const bool end = rank_of[u] == stays - 1;
                bool cuts;  // the token is the last one that stays
                if constexpr (kCount) cuts = top_p < 1.0 ? rank_of[u] < stays && (rank_of[u] == 0 || from < target) && (end || to >= target) : end;
                else cuts = above + from * 0x1p-52 < target && above + to * 0x1p-52 >= target;
                if (cuts) sh.verdict = sh.list[t];
            }
            __syncthreads();
            return sh.verdict;
        }
        int size = 2 * kPairs;
        while (size < static_cast<int>(n)) size *= 2;
        const int t = threadIdx.x;
        for (int i = t; i < size; i += NT)
            if (i >= static_cast<int>(n)) sh.list[i] = 0;
        for (int k = 2; k <= size; k *= 2)  // bitonic
            for (int j = k / 2; j > 0; j /= 2) {
                __syncthreads();
                for (int u = t; u < size / 2; u += NT) {
                    const int i = 2 * u - (u & (j - 1));
                    const unsigned long long p = sh.list[i], q = sh.list[i + j];
                    if ((p < q) == ((i & k) == 0)) {
                        sh.list[i] = q;
                        sh.list[i + j] = p;
                    }
                }
            }
        __syncthreads();
        int last = static_cast<int>(kCount ? min(want, n) : n) - 1;
        if (!kCount || top_p < 1.0) {
            constexpr int kOwn = kList / NT;
            double w[kOwn], mine = 0.0;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const int i = kOwn * t + j;
                w[j] = i <= last ? weight(value_of(static_cast<uint32_t>(sh.list[i] >> 32))) : 0.0;
                mine += w[j];
            }
            double upto = warp_upto(mine, lane), all = 0.0;
            if (lane == 31) sh.scan[warp] = upto;
            if (t == 0) sh.last = kCount ? last : kList;
            __syncthreads();
            for (int q = 0; q < kWarps; ++q) {
                if (q < warp) upto += sh.scan[q];
                all += sh.scan[q];
            }
            if (kCount) target = top_p * all;
            upto += above - mine;
            for (int j = 0; j < kOwn; ++j) {
                upto += w[j];
                if (kOwn * t + j <= last && upto >= target) {
                    atomicMin(&sh.last, kOwn * t + j);
                    break;
                }
            }
            __syncthreads();
            last = sh.last;
            if (last == kList) return 0;
        }
        return sh.list[last];
    }

    // Rank 0: the draw from n listed tokens, those up to the cut; four threads a token, as in cut_of_list().
    __device__ __forceinline__ void draw_listed(uint32_t n, unsigned long long cut, float uniform, int64_t row) {
        const int q = threadIdx.x & 3;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += NT) sh.part[i] = sh.list[i] >= cut ? units_of(sh.list[i]) : 0;
        __syncthreads();
#pragma unroll 1
        for (uint32_t t0 = 0; t0 < n; t0 += NT / 4) {
            const uint32_t t = t0 + threadIdx.x / 4;
            const unsigned long long mine = t < n ? sh.list[t] : 0, own = t < n ? sh.part[t] : 0;
            unsigned long long before = 0, all = 0;
            for (uint32_t j = q; j < n; j += 4) {
                all += sh.part[j];
                before += static_cast<uint32_t>(sh.list[j]) > static_cast<uint32_t>(mine) ? sh.part[j] : 0;  // a lower index
            }
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                before += __shfl_xor_sync(kAll, before, o);
                all += __shfl_xor_sync(kAll, all, o);
            }
            const double target = (uniform > 0.0f ? static_cast<double>(uniform) : 0.0) * static_cast<double>(all);
            if (q == 0 && own > 0 && static_cast<double>(before) <= target && (static_cast<double>(before + own) > target || before + own == all)) {
                a.tokens[row] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(mine));
                if (a.logprob != nullptr) a.logprob[row] = static_cast<float>(log(weight(value_of(static_cast<uint32_t>(mine >> 32))) / (static_cast<double>(all) * 0x1p-52)));
            }
        }
    }

    // The first k tokens' cut (0: there are fewer, all stay). own: the thread's largest logit, low: the least
    // of these that counts, least: a bound of all that do. Where the first k are few, top_p (below 1) is
    // applied to them too, and listed is how many are in the list, all that stay among them.
    __device__ __forceinline__ unsigned long long cut_count(float own, float low, float least, float best, uint32_t k, double top_p, uint32_t &listed) {
        float lo = least;
        if (k <= static_cast<uint32_t>(a.ctas) * (NT / 2)) {
            // k threads' largest logits are k tokens at or above their bin's lower edge
            set_bins(low, best);
            clear_bins();
            if (own >= low) atomicAdd(&sh.bins[bin(own)], 1u);
            cluster_sync_all();
            const int star = find_bin(k);
            if (star < kBins) lo = fmaxf(least, edge_below(star, low));
            uint32_t count = 0;
            pick([&](float v, int) { return v >= lo; }, [&](float y, int j, bool is) {
                list(y, j, is, 0);
                count += is;
            });
            listed = count_of(tell(0, __reduce_add_sync(kAll, count)));
            if (listed <= kList) {
                const unsigned long long c = cut_of_list<true>(listed, k, 0.0, 0.0, top_p);
                return listed < k && !(top_p < 1.0) ? 0ull : c;
            }
        }
        listed = kList + 1;
        return slowly<true>([](float, int) { return true; }, lo, best, k, 0.0, 0.0);
    }

    // The cut of the fewest first tokens, of those that `keep` takes (all, but for `some`), whose weights sum to
    // top_p of theirs. above: what the warp's tokens before the list sum to (all_listed: there are none), listed:
    // the tokens in the list (more than kList: neither holds). A bin that more than 2^17 tokens of a CTA share
    // may wrap: the exact sums then say that the cut is not there.
    template <typename F>
    __device__ __forceinline__ unsigned long long cut_mass(F keep, bool some, float least, double top_p, double &above, uint32_t &listed, bool &all_listed) {
        clear_bins();
        double mass = 0.0;
        auto weigh = [&](const float(&v)[E], int i, auto some) {
            double w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = weight(v[e]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool in = !decltype(some)::value || keep(v[e], i + e);
                mass += in ? w[e] : 0.0;
                // 64 bins to a factor of two by the upper bits of w; in units of 2^-14 of that power
                const uint32_t high = __double2hiint(w[e]), b = (kOneBits >> kBinShift) - (high >> kBinShift);
                if (in && weight.counts(v[e]) && b < kBins) atomicAdd(&sh.bins[b], ((high & 0xfffffu) | 0x100000u) >> 6);
            }
        };
        if (some) sweep([&](const float(&v)[E], int i) { weigh(v, i, std::true_type{}); });
        else sweep([&](const float(&v)[E], int i) { weigh(v, i, std::false_type{}); });
        const double whole = sum_of(tell(__double_as_longlong(warp_sum(mass)), 0)), target = top_p * whole;
        // the bins before which the sum, 1e-4 of the whole more or less, does not reach the target
        {
            float c[kPer], mine = 0.0f, tokens = 0.0f;  // mass, and at most so many tokens (a unit sum is 2^14 to 2^15 each)
            all_bins(c);
            const int b = kPer * threadIdx.x;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                tokens += c[j] * 0x1p-14f;
                c[j] *= __int_as_float((127 - 14 - (b + j + 63) / 64) << 23);
                mine += c[j];
            }
            float upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float y = __shfl_up_sync(kAll, upto, o);
                if (lane >= o) upto += y;
            }
            if (lane == 31) sh.scan_f[warp] = upto;
            __syncthreads();
            float before = lane < warp ? sh.scan_f[lane] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(kAll, before, o);
            upto += before - mine;
            const float low = static_cast<float>(target - 1e-4 * whole), high = static_cast<float>(target + 1e-4 * whole);
            int first = kBins, last = kBins;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                upto += c[j];
                if (first == kBins && upto >= low) first = b + j;
                if (last == kBins && upto >= high) last = b + j;
            }
            if (first < kBins) atomicMin(&sh.first, first);
            if (last < kBins) atomicMin(&sh.last, last);
            __syncthreads();
            // few tokens up to the last of these bins: they are all listed
            tokens = b <= min(sh.last, kBins - 2) ? tokens : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) tokens += __shfl_xor_sync(kAll, tokens, o);
            if (lane == 0) sh.scan_f[warp] = tokens;
            __syncthreads();
            tokens = lane < kWarps ? sh.scan_f[lane] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) tokens += __shfl_xor_sync(kAll, tokens, o);
            all_listed = tokens <= kPairs;
        }
        const int first = sh.first, last = min(sh.last, kBins - 2);
        listed = kList + 1;
        if (first < kBins - 1) {
            // what lies before them, exactly, and their tokens
            const float from = all_listed ? INFINITY : edge_above(first), to = edge_above(last + 1);
            uint32_t count = 0;
            double sum = 0.0;
            pick([&](float v, int i) { return v >= to && (!some || keep(v, i)); }, [&](float y, int j, bool is) {
                list(y, j, is && y <= from, 1);
                count += is && y <= from;
                if (all_listed) return;
                const double w = weight(y);
                sum += is && y > from ? w : 0.0;
            });
            above = warp_sum(sum);
            const Told got = tell(__double_as_longlong(above), __reduce_add_sync(kAll, count));
            const double all_above = sum_of(got);
            const uint32_t k = count_of(got);
            if (k <= kList && all_above < target) {
                const unsigned long long c = cut_of_list<false>(k, 0, all_above, target, 1.0);
                if (c != 0) {
                    listed = k;
                    return c;
                }
            }
        }
        // The tokens lighter than (1 - top_p) of the mean weight weigh less than 1 - top_p together: the cut is above them.
        const double t = log2((1.0 - top_p) * whole / a.vocab) / weight.per;
        const double margin = 1e-6 * (fabs(weight.top) + fabs(t));
        return slowly<false>(keep, fmaxf(least, static_cast<float>(fmax(weight.top + t - margin, kLowest))), static_cast<float>(weight.top), 0, target, whole);
    }

    // cut_slow() apart, on a copy: its registers are not the quick ways' concern.
    template <bool kCount, typename F>
    __device__ __forceinline__ unsigned long long slowly(F inside, float lo, float to, uint32_t want, double target, double whole) {
        Row copy = *this;
        const unsigned long long c = copy.template cut_slow<kCount>(inside, lo, to, want, target, whole);
        turn = copy.turn;
        return c;
    }
    // The cut of the first `want` tokens that `inside` takes (kCount; 0: there are fewer), or of the fewest
    // first ones whose weights sum to `target`, in steps: a histogram of the range, the
    // part before its bin and that bin, and the range that holds the cut again, until it
    // fits the list or is one value. For what the quick ways do not find (many equal logits,
    // large top_k, a cut 32 factors of two below the largest weight).
    template <bool kCount, typename F>
    __device__ __noinline__ unsigned long long cut_slow(F inside, float lo, float to, uint32_t want, double target, double whole) {
        double above = 0.0, range_mass = whole;
        while (true) {
            cluster_sync_all();  // the list's count and the bins have been read
            // shares of the range's mass in 32 bits, at least 1 of each token
            const float unit = kCount ? 0.0f : static_cast<float>(2147483648.0 / range_mass);
            set_bins(lo, to);
            if (threadIdx.x == 0) sh.listed[0] = 0;
            clear_bins();
            sweep([&](const float(&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (v[e] >= lo && v[e] <= to && inside(v[e], i + e))
                        atomicAdd(&sh.bins[bin(v[e])], kCount ? 1u : max(1u, __float2uint_rn(exp2f((v[e] - static_cast<float>(weight.top)) * static_cast<float>(weight.per)) * unit)));
            });
            cluster_sync_all();
            const double share = kCount ? 0.0 : (target - above) / range_mass * 2147483648.0;
            int star = find_bin(kCount ? want : (share < 1.0 ? 1u : static_cast<uint32_t>(fmin(share, 4294967295.0))));
            if (kCount && star == kBins) {
                cluster_sync_all();  // the bins have been read
                return 0;
            }
            const int filled = sh.filled;
            star = min(star, filled);
            if (kCount) want -= sh.under;
            // the mass before this bin, its tokens into the list, and what bounds the three ranges
            float low0 = INFINITY, low1 = INFINITY, high1 = -INFINITY, high2 = -INFINITY;
            uint32_t count = 0;
            double sum = 0.0;
            pick([&](float v, int i) { return v >= lo && v <= to && inside(v, i); }, [&](float y, int j, bool is) {
                const int at = is ? bin(y) : kBins;
                list(y, j, at == star, 0);
                if (at < star) {
                    low0 = fminf(low0, y);
                    if (!kCount) sum += weight(y);
                } else if (at == star) {
                    low1 = fminf(low1, y);
                    high1 = fmaxf(high1, y);
                    ++count;
                } else if (is) {
                    high2 = fmaxf(high2, y);
                }
            });
            const Told got = tell(__double_as_longlong(warp_sum(sum)), __reduce_add_sync(kAll, count));
            const double before = kCount ? 0.0 : sum_of(got);
            const uint32_t listed = count_of(got);
            int range_of = 1;  // in which of the three the cut lies
            if (!kCount && above + before >= target && before > 0.0) {
                range_of = 0;
                range_mass = before;
            } else {
                above += before;
                if (listed <= kList) {
                    // behind the list only where there is something
                    const unsigned long long c = cut_of_list<kCount>(listed, want, above, target, 1.0);
                    if (c != 0) return c;
                }
                if constexpr (!kCount) {
                    const double within = sum_of(tell(__double_as_longlong(mass_of([&](float v, int i) { return v >= lo && v <= to && bin(v) == star && inside(v, i); })), 0));
                    if (filled > star && above + within < target) {
                        range_of = 2;
                        above += within;
                        range_mass = whole - above;
                    } else {
                        range_mass = within;
                        if (listed <= kList) return entry_of(lowest(low1), 0x7fffffff);  // the last of all, short of the target by a rounding
                    }
                }
            }
            range_mass = fmax(range_mass, 1e-9 * whole);  // the shares' sum stays within 32 bits whatever the differences' rounding
            const float most = range_of == 0 ? to : (range_of == 1 ? high1 : high2), least = range_of == 0 ? low0 : (range_of == 1 ? low1 : lo);
            const Told ends = tell(__reduce_max_sync(kAll, key_of(most + 0.0f)), __reduce_max_sync(kAll, 0xffffffffu - key_of(least + 0.0f)));
            to = value_of(largest(ends, 0, 0));
            lo = value_of(0xffffffffu - largest(ends, 1, 0));
            if (lo >= to) {
                uint32_t r = want;
                if constexpr (!kCount) {
                    const double w = weight(to);
                    uint32_t short_of = 0;  // the least number of them that reaches the target
                    r = static_cast<uint32_t>(a.vocab);
                    while (r - short_of > 1) {
                        const uint32_t mid = short_of + (r - short_of) / 2;
                        if (above + mid * w >= target) r = mid;
                        else short_of = mid;
                    }
                }
                return entry_of(to, nth_equal(to, r, inside));
            }
        }
    }
    __device__ __forceinline__ float lowest(float v) {  // of the row's threads
        return value_of(0xffffffffu - largest(tell(__reduce_max_sync(kAll, 0xffffffffu - key_of(v + 0.0f)), 0), 0, 0));
    }

    // The index of the r-th token (from 1; past the last: that) of logit x that `inside` takes, by rising index.
    template <typename F>
    __device__ __forceinline__ int nth_equal(float equal, uint32_t r, F inside) {
        const int n = steps();
        auto marks = [&](int s) {
            float v[E];
            load(s, v);
            const int i = index_of(s);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c |= v[e] == equal && inside(v[e], i + e) ? 1u << e : 0u;
            return c;
        };
        uint32_t mine = 0;
        for (int s = 0; s < n; ++s) mine += __popc(marks(s));
        mine = __reduce_add_sync(kAll, mine);
        const Told got = tell(mine, 0);
        uint32_t before = 0, all = 0;
        for (int q = 0; q < a.ctas * kWarps; ++q) {
            if (q < rank * kWarps + warp) before += static_cast<uint32_t>(got[q][0]);
            all += static_cast<uint32_t>(got[q][0]);
        }
        r = min(r, all);
        if (r > before && r <= before + mine) {
            uint32_t left = r - before;
            for (int s = 0; s < n; ++s) {
                const uint32_t c = marks(s), k = __popc(c);
                uint32_t upto = k;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(kAll, upto, o);
                    if (lane >= o) upto += y;
                }
                const uint32_t in_step = __shfl_sync(kAll, upto, 31);
                if (left > in_step) {
                    left -= in_step;
                    continue;
                }
                if (left <= upto && left > upto - k) {
                    uint32_t m = c;
                    for (uint32_t q = left - (upto - k); q > 1; --q) m &= m - 1;
                    const int found = index_of(s) + __ffs(m) - 1;
                    for (int q = 0; q < a.ctas; ++q) st_cluster(mapa_shared(smem_u32(&sh.verdict), q), static_cast<unsigned long long>(found));
                }
                break;
            }
        }
        cluster_sync_all();
        return static_cast<int>(sh.verdict);
    }
};

template <typename T, bool STAGED, int NT>
__global__ void __launch_bounds__(NT, NT == 1024 ? 1 : 3) k_sample(SampleArgs a) {
    constexpr int kWarps = NT / 32;
    extern __shared__ __align__(16) uint8_t dyn[];
    Shared<NT> &sh = *reinterpret_cast<Shared<NT> *>(dyn);
    using R = Row<T, STAGED, NT>;
    griddep_launch_dependents();
    const int64_t row = blockIdx.x / a.ctas;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    R r{a, sh, reinterpret_cast<T *>(dyn + kShared<NT>), x, static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)), static_cast<int>(blockIdx.x % a.ctas),
        static_cast<int>(threadIdx.x & 31), static_cast<int>(threadIdx.x >> 5)};
    if (threadIdx.x < 2) sh.listed[threadIdx.x] = 0;
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    griddep_wait();
    const float temperature = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    const int top_k = a.top_k != nullptr ? a.top_k[row] : 0;
    const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f, min_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    const float uniform = a.uniform[row];

    // the row into shared memory, and its largest
    float own = -INFINITY, best = -INFINITY, low = -INFINITY;  // low: the least of the threads' largest
    double per;
    int best_at = -1;
    {
        int own_at = 0x7fffffff;
        constexpr int kAhead = R::kAhead;
        const int n = r.steps();
#pragma unroll 1
        for (int s0 = 0; s0 < n; s0 += kAhead) {
            alignas(16) T t[kAhead][R::E];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (s0 + j < n) r.fetch(s0 + j, t[j]);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (s0 + j >= n) break;
                if constexpr (STAGED) *reinterpret_cast<uint4 *>(r.staged(s0 + j)) = *reinterpret_cast<const uint4 *>(t[j]);
                const int i = r.index_of(s0 + j);
#pragma unroll
                for (int e = 0; e < R::E; ++e) {
                    const float v = Elem<T>::load(t[j] + e);
                    if (v > own) {  // NaN is not
                        own = v;
                        own_at = i + e;
                    }
                }
            }
        }
        const uint32_t key = own_at != 0x7fffffff ? key_of(own + 0.0f) : 0u, most = __reduce_max_sync(kAll, key);
        const int first = __reduce_min_sync(kAll, key == most ? own_at : 0x7fffffff);
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every CTA has started
        r.say(static_cast<unsigned long long>(most) << 32 | (0xffffffffu - static_cast<uint32_t>(first)),
              __reduce_max_sync(kAll, key != 0 ? 0xffffffffu - key : 0u));
        per = 1.4426950408889634074 / temperature;  // while the others arrive
        const auto got = r.hear();
        const uint32_t top = r.largest(got, 0, 1);
        if (top != 0) {
            best = value_of(top);
            uint32_t at = 0;
            for (int i = r.lane; i < a.ctas * kWarps; i += 32) at = max(at, got[i][0] >> 32 == top ? static_cast<uint32_t>(got[i][0]) : 0u);
            best_at = static_cast<int>(0xffffffffu - __reduce_max_sync(kAll, at));
        }
        low = value_of(0xffffffffu - r.largest(got, 1, 0));
    }
    if (best_at < 0 || best == INFINITY || !(temperature > 0.0f) || top_k == 1 || top_p <= 0.0f) {
        if (r.rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = best_at;
            if (a.logprob != nullptr) a.logprob[row] = best_at < 0 ? NAN : 0.0f;
        }
        return;
    }
    // 2^-1000. Rounded up: to nearest it may lie half a float's spacing lower, which at a small
    // temperature is far more than the exponents that a weight has below 2^-1000.
    const float least = fmaxf(__fsub_ru(best, 693.147f * temperature), kLowest);
    r.weight = Weight{best, per, least};
    const Weight &weight = r.weight;

    // the cut: kept are the tokens up to it in the order
    unsigned long long cut = 0;
    float cut_x = -INFINITY;
    int cut_i = 0x7fffffff;
    auto keep = [&](float v, int i) { return v > cut_x || (v == cut_x && i <= cut_i); };
    auto set_cut = [&](unsigned long long c) {
        if (c <= cut) return;
        cut = c;
        cut_x = value_of(static_cast<uint32_t>(c >> 32));
        cut_i = static_cast<int>(0xffffffffu - static_cast<uint32_t>(c));
    };
    const bool has_k = top_k > 0 && top_k < a.vocab, has_p = top_p < 1.0f;
    uint32_t listed = kList + 1;  // where it is less, the kept tokens are in the list, but for those that `above` sums
    double above = 0.0;
    bool all_listed = true;
    if (has_k) set_cut(r.cut_count(own, fmaxf(low, least), least, best, static_cast<uint32_t>(top_k), has_p ? static_cast<double>(top_p) : 1.0, listed));
    if (has_p && listed > kList) {
        const float cx = cut_x;
        const int ci = cut_i;
        set_cut(r.cut_mass([=](float v, int i) { return v > cx || (v == cx && i <= ci); }, cut != 0, fmaxf(least, cx), static_cast<double>(top_p), above, listed, all_listed));
    }
    if (min_p > 0.0f) {
        // The least float whose weight is min_p or more: of 32 about the logarithm's, or where it is not among
        // them (weights round to min_p over many floats: a largest logit near 0), by halving.
        const double at_least = min_p < 1.0f ? min_p : 1.0;
        const uint32_t k_top = key_of(best), about = key_of(fmaxf(best + log2f(static_cast<float>(at_least)) / static_cast<float>(per), kLowest) + 0.0f);
        uint32_t k = min(about + 8, k_top) - 31 + r.lane;
        const uint32_t reach = __ballot_sync(kAll, weight(value_of(k)) >= at_least);
        if ((reach & 1u) == 0 && reach != 0) {
            k = __shfl_sync(kAll, k, __ffs(reach) - 1);
        } else {
            uint32_t under = key_of(kLowest) - 1;
            k = k_top;
            while (k - under > 1) {
                const uint32_t mid = under + (k - under) / 2;
                if (weight(value_of(mid)) >= at_least) k = mid;
                else under = mid;
            }
        }
        const unsigned long long c = static_cast<unsigned long long>(k) << 32 | (0xffffffffu - 0x7fffffffu);
        if (c > cut) {
            set_cut(c);
            if (!all_listed) listed = kList + 1;  // it may lie among the tokens that `above` sums
        }
    }

    // the draw: from the list, if that is short and all there is
    if (listed <= kPairs && all_listed) {
        if (r.rank == 0) r.draw_listed(listed, cut, uniform, row);
        return;
    }
    double mass;
    if (listed <= kList) {
        mass = 0.0;
        if (listed <= kPairs) {  // in no fixed order: as whole numbers
            unsigned long long sum = 0;
            for (uint32_t j = r.lane; j < listed; j += 32) {
                const unsigned long long e = sh.list[j];
                const float v = value_of(static_cast<uint32_t>(e >> 32));
                const int i = static_cast<int>(0xffffffffu - static_cast<uint32_t>(e));
                if (r.own_warp(i) && keep(v, i)) sum += r.units_of(e);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
            mass = static_cast<double>(sum) * 0x1p-52;
        } else {
            for (uint32_t j = r.lane; j < listed; j += 32) {
                const unsigned long long e = sh.list[j];
                const float v = value_of(static_cast<uint32_t>(e >> 32));
                const int i = static_cast<int>(0xffffffffu - static_cast<uint32_t>(e));
                if (r.own_warp(i) && keep(v, i)) mass += weight(v);
            }
            mass = warp_sum(mass);
        }
        mass += above;
    } else {
        mass = cut == 0 ? r.mass_of_all() : r.mass_of(keep);
    }
    const auto parts = r.tell(__double_as_longlong(mass), 0);
    // each lane takes the same number of warps, in the order of the tokens
    const int count = a.ctas * kWarps, each = (count + 31) / 32;
    double sum_here = 0.0;
    for (int q = r.lane * each; q < min((r.lane + 1) * each, count); ++q) sum_here += __longlong_as_double(parts[q][0]);
    const double upto = warp_upto(sum_here, r.lane), sum = __shfl_sync(kAll, upto, 31);
    const double target = (uniform > 0.0f ? static_cast<double>(uniform) : 0.0) * sum;
    // the first warp that passes the target, else the last that holds anything
    int owner = -1;
    bool passed_here = false;
    double at_warp = upto - sum_here, before = at_warp;
    for (int q = r.lane * each; q < min((r.lane + 1) * each, count) && !passed_here; ++q) {
        const double m = __longlong_as_double(parts[q][0]);
        if (m > 0.0) {
            owner = q;
            at_warp = before;
            passed_here = before + m > target;
        }
        before += m;
    }
    const uint32_t passing = __ballot_sync(kAll, passed_here), holding = __ballot_sync(kAll, owner >= 0);
    const int from = passing != 0 ? __ffs(passing) - 1 : 31 - __clz(holding);
    owner = __shfl_sync(kAll, owner, from);
    at_warp = __shfl_sync(kAll, at_warp, from);
    if (owner < 0) {  // no warp holds anything; the largest logit weighs 1, so no row comes here, and none would go without a token
        if (r.rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = best_at;
            if (a.logprob != nullptr) a.logprob[row] = 0.0f;
        }
        return;
    }
    if (owner / kWarps != r.rank) return;
    // The owner's CTA: a warp per step of the owner's tokens finds the one that passes, else the last that holds anything.
    r.warp = owner % kWarps;
    const int n = r.steps(), me = threadIdx.x >> 5;
    int step = -1;
    double at_step = at_warp;
    for (int s0 = 0; s0 < n; s0 += kWarps) {
        double m = 0.0;
        if (s0 + me < n) {
            float v[R::E];
            r.load(s0 + me, v);
            const int i = r.index_of(s0 + me);
#pragma unroll
            for (int e = 0; e < R::E; ++e) {
                const double w = weight(v[e]);
                m += keep(v[e], i + e) ? w : 0.0;
            }
        }
        m = warp_sum(m);
        __syncthreads();
        if (r.lane == 0) sh.scan[me] = m;
        __syncthreads();
        m = r.lane < kWarps ? sh.scan[r.lane] : 0.0;
        const double to = at_warp + warp_upto(m, r.lane);
        const uint32_t passed = __ballot_sync(kAll, m > 0.0 && to > target), holds = __ballot_sync(kAll, m > 0.0);
        if (holds != 0) {
            const int l = passed != 0 ? __ffs(passed) - 1 : 31 - __clz(holds);
            step = s0 + l;
            at_step = __shfl_sync(kAll, to - m, l);
        }
        if (passed != 0) break;
        at_warp = __shfl_sync(kAll, to, 31);
    }
    if (me != 0) return;
    // its lane, and the lane's token
    int found = -1;
    double found_w = 0.0;
    {
        float v[R::E];
        r.load(step, v);
        const int i = r.index_of(step);
        double w[R::E], mine = 0.0;
#pragma unroll
        for (int e = 0; e < R::E; ++e) {
            w[e] = weight(v[e]);
            w[e] = keep(v[e], i + e) ? w[e] : 0.0;
            mine += w[e];
        }
        const double to = at_step + warp_upto(mine, r.lane);
        const uint32_t passed = __ballot_sync(kAll, to > target && mine > 0.0), holds = __ballot_sync(kAll, mine > 0.0);
        if (r.lane == (passed != 0 ? __ffs(passed) - 1 : 31 - __clz(holds))) {
            double c = to - mine;
#pragma unroll
            for (int e = 0; e < R::E; ++e) {
                if (w[e] > 0.0 && !(found >= 0 && c > target)) {
                    found = i + e;
                    found_w = w[e];
                    c += w[e];
                }
            }
        }
    }
    const int token = __reduce_max_sync(kAll, found);
    if (found == token && token >= 0) {
        a.tokens[row] = token;
        if (a.logprob != nullptr) a.logprob[row] = static_cast<float>(log(found_w / sum));
    }
}

template <typename T, bool STAGED, int NT>
int launch_sample(const SampleArgs &a, int64_t rows, cudaStream_t st) {
    auto kern = k_sample<T, STAGED, NT>;
    const int smem = kShared<NT> + (STAGED ? a.slice * static_cast<int>(sizeof(T)) : 0);
    const int rc = ensure_max_smem(reinterpret_cast<const void *>(kern), kShared<NT> + kStageMost<NT>, "sample");
    if (rc != LCML_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * a.ctas));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(a.ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(LCML_ERR_CUDA, "sample launch failed: %s", cudaGetErrorString(e));
    }
    return LCML_OK;
}

template <typename T>
int dispatch_sample(SampleArgs a, int64_t rows, cudaStream_t st) {
    LCML_CHECK_ARG(rows <= 0x7fffffff / kMaxCluster, "lcml_sample: too many rows for one call");
    constexpr int E = Row<T, true, 1024>::E;
    const int64_t length = static_cast<int64_t>(a.vocab) + E - 1;
    auto slice = [&](int ctas, int threads) {
        const int64_t unit = static_cast<int64_t>(threads) * E * ctas;
        return (length + unit - 1) / unit * threads * E;
    };
    // CTAs of 256 threads where they hold few tokens (a row of 2000 with top_p in two of them 13.8 us, 15.3 in
    // two of 1024; 8 of 10000 with top_k 100 11.6 and 13.0), else of 1024, one an SM.
    // Several CTAs a row while each finds an SM and keeps 16384 tokens: 16 rows of 128001 with top_p 0.9
    // take 74 us in one each, 47 in two, 35 in four; in eight 62, as clusters of so many find no
    // room beside each other. 36 rows 74, 47 and, no longer all at once, 64.
    auto fits = [&](int ctas) { return rows * ctas <= sm_count() * 7 / 8; };
    const int few = fits(2) ? 2 : 1;
    if (a.vocab <= few * few * 4096) {
        a.ctas = few;
        a.slice = static_cast<int>(slice(few, 256));
        return launch_sample<T, true, 256>(a, rows, st);
    }
    while (a.ctas < kMaxCluster && fits(2 * a.ctas) && slice(a.ctas, 1024) > 16384) a.ctas *= 2;
    a.slice = static_cast<int>(slice(a.ctas, 1024));
    if (a.slice * static_cast<int64_t>(sizeof(T)) > kStageMost<1024>) return launch_sample<T, false, 1024>(a, rows, st);
    return launch_sample<T, true, 1024>(a, rows, st);
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" int lcml_sample(const lcml_sample_desc *d, lcml_stream_t stream) {
    LCML_CHECK_ARG(d != nullptr, "lcml_sample: null descriptor");
    LCML_CHECK_ARG(d->rows >= 0 && d->vocab >= 0, "lcml_sample: negative extent");
    LCML_CHECK_ARG(d->dtype == LCML_DTYPE_FLOAT || d->dtype == LCML_DTYPE_FLOAT16 || d->dtype == LCML_DTYPE_BFLOAT16, "lcml_sample: dtype %d unsupported", d->dtype);
    if (d->rows == 0) return LCML_OK;
    LCML_CHECK_ARG(d->vocab > 0, "lcml_sample: rows without tokens");
    LCML_CHECK_ARG(d->vocab <= 0x7fffffff - 65536, "lcml_sample: vocab is too large");
    LCML_CHECK_ARG(d->logits && d->uniform && d->tokens, "lcml_sample: null pointer");
    LCML_CHECK_ARG(d->ld >= d->vocab || d->rows == 1, "lcml_sample: ld is less than vocab %lld", (long long)d->vocab);
    const uintptr_t es = d->dtype == LCML_DTYPE_FLOAT ? 4 : 2;
    LCML_CHECK_ARG(aligned(d->logits, es) && aligned(d->uniform, 4) && aligned(d->temperature, 4) && aligned(d->top_k, 4) && aligned(d->top_p, 4) && aligned(d->min_p, 4) &&
                       aligned(d->tokens, 4) && aligned(d->logprob, 4),
                   "lcml_sample: a pointer is not aligned to its element size");
    const SampleArgs a{d->logits, d->ld, static_cast<int>(d->vocab), 0, 1, d->uniform, d->temperature, d->top_k, d->top_p, d->min_p, d->tokens, d->logprob};
    cudaStream_t st = to_cuda(stream);
    if (d->dtype == LCML_DTYPE_FLOAT) return dispatch_sample<float>(a, d->rows, st);
    if (d->dtype == LCML_DTYPE_FLOAT16) return dispatch_sample<__half>(a, d->rows, st);
    return dispatch_sample<__nv_bfloat16>(a, d->rows, st);
}
