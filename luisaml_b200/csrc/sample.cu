// The next token of every row of logits (lcml_sample): temperature, top-k, top-p,
// min-p, then the draw from a given uniform number.
//
// One cluster of CTAs per row; the row is read once and stays in the cluster's
// shared memory (rows too long for that are read again from L2). What top-k,
// top-p and min-p keep is a prefix of the tokens by falling logit, so each comes
// down to its last token, the cut (x, index). No sort finds it:
//   1. a histogram of the tokens between two bounds of the cut, counts only. A
//      bin's count times the weight at its middle is about its mass, which says
//      in which bin the kept mass should pass its target (for top-k: does).
//   2. the mass above that bin and in it, with as many neighbours as the list
//      holds, exactly; their tokens into the list, which one CTA sorts and sums to
//      find the cut. Where the cut lies above or below after all, or the bin is
//      too full, that range is binned again, until it fits or all of it is one
//      value: then the cut is the r-th of them by index.
// The draw needs no order either: weights of the kept tokens summed by rising
// index, per warp, then the warp that holds uniform * sum goes over its tokens
// once more.
//
// Weights and sums are fp64, in an order that the sizes fix: a token lies within
// an fp32 rounding of its neighbours' range once in some thousand rows, and the
// result would go by the order of the sum. The weight is 2^t with a polynomial of
// 8e-13; its fp64 instructions run at half the fp32 rate.
#include "lcml_decoder.cuh"

#include "../../include/lcml_decode_step.h"

namespace lcml {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 2 * kThreads;
constexpr int kList = 2 * kThreads;  // tokens that one CTA sorts
constexpr unsigned kAll = 0xffffffffu;

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

struct Shared {
    unsigned long long slot[2][kMaxCluster][2];  // what the row's CTAs tell each other, two turns
    unsigned long long red[2][kWarps];
    double mass[kWarps];
    unsigned long long list[kList];
    uint32_t bins[kBins];
    double scan[2][kWarps];
    int star, filled, from, to;  // the bin where the cut should lie, the last one that holds anything, the bins looked at
    uint32_t star_first, star_last, skipped, reached, all;  // tokens before and up to the bin, before and up to these bins, in all
    int last;
    unsigned long long verdict;  // the cut, from the CTA that finds it
    uint32_t listed;
};

// Order-preserving bits of a float (no NaN).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A token in the order: falling logit, equal ones by rising index.
__device__ __forceinline__ unsigned long long entry_of(float x, int index) {
    return static_cast<unsigned long long>(key_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

struct Weight {
    double top, per;  // largest logit, log2(e) / temperature
    // 2^((x - top) per): the exponent's nearest whole number by addition of 1.5 2^52, 2^f
    // on [-1/2, 1/2] as 1 + f p(f), p fitted at Chebyshev points with 2^f's relative
    // error as the weight (8.2e-13), so the largest logit has exactly 1.
    __device__ __forceinline__ double operator()(float x) const {
        const double t = (static_cast<double>(x) - top) * per;
        const double s = t + 6755399441055744.0;
        const double f = t - (s - 6755399441055744.0);
        double p = 1.3178918944060163e-06;
        p = fma(p, f, 1.5309155627301653e-05);
        p = fma(p, f, 0.00015403825519790757);
        p = fma(p, f, 0.0013333454862616348);
        p = fma(p, f, 0.009618128616057417);
        p = fma(p, f, 0.055504109352640572);
        p = fma(p, f, 0.24022650698110781);
        p = fma(p, f, 0.69314718054821356);
        p = fma(p, f, 1.0);
        const double w = __hiloint2double(__double2hiint(p) + (__double2loint(s) << 20), __double2loint(p));
        return t > -1000.0 ? w : 0.0;  // NaN (an infinite temperature and -infinity) too
    }
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

template <typename T, bool STAGED>
struct Row {
    static constexpr int E = 16 / static_cast<int>(sizeof(T));  // tokens a lane takes at once
    static constexpr int kStep = 32 * E;

    const SampleArgs &a;
    Shared &sh;
    T *stage;        // the CTA's slice
    const T *x;      // the row
    int off;         // tokens by which the row begins after a 16-byte boundary
    int rank, lane, warp;
    int turn = 0;
    Weight weight;

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
    __device__ __forceinline__ void fetch(int s, T (&t)[E]) const {
        const int i = index_of(s);
        if (i >= 0 && i + E <= a.vocab) {
            *reinterpret_cast<uint4 *>(t) = __ldg(reinterpret_cast<const uint4 *>(x + i));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] = i + e >= 0 && i + e < a.vocab ? x[i + e] : Elem<T>::from(-INFINITY);
        }
    }
    __device__ __forceinline__ void clean(const T (&t)[E], float (&v)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float f = Elem<T>::load(t + e) + 0.0f;  // -0 is 0
            v[e] = f == f ? f : -INFINITY;
        }
    }
    __device__ __forceinline__ T *staged(int s) const { return stage + warp * (a.slice / kWarps) + s * kStep + lane * E; }
    __device__ __forceinline__ void load(int s, float (&v)[E]) const {
        alignas(16) T t[E];
        if constexpr (STAGED) *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(staged(s));
        else fetch(s, t);
        clean(t, v);
    }

    // Exchange of two values per CTA; every thread gets all of them in sh.slot[..].
    __device__ __forceinline__ const unsigned long long (*tell(unsigned long long v0, unsigned long long v1))[2] {
        if (threadIdx.x < a.ctas) {
            const uint32_t to = mapa_shared(smem_u32(&sh.slot[turn][rank][0]), threadIdx.x);
            st_cluster(to, v0);
            st_cluster(to + 8, v1);
        }
        cluster_sync_all();
        const auto *got = sh.slot[turn];
        turn ^= 1;
        return got;
    }
    template <typename F>
    __device__ __forceinline__ unsigned long long block_reduce(unsigned long long v, int which, F op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
        __syncthreads();
        if (lane == 0) sh.red[which][warp] = v;
        __syncthreads();
        v = sh.red[which][0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v = op(v, sh.red[which][w]);
        return v;
    }

    // Sum of the weights of the tokens that `keep` takes: per warp in sh.mass, and over the row.
    template <typename F>
    __device__ __forceinline__ double mass_of(F keep) {
        double sum = 0.0;
        const int n = steps();
        for (int s = 0; s < n; ++s) {
            float v[E];
            load(s, v);
            uint32_t in = 0;
            const int i = index_of(s);
#pragma unroll
            for (int e = 0; e < E; ++e) in |= keep(v[e], i + e) ? 1u << e : 0u;
            if (!__any_sync(kAll, in != 0)) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double w = weight(v[e]);
                sum += in >> e & 1u ? w : 0.0;
            }
        }
        sum = warp_sum(sum);
        __syncthreads();
        if (lane == 0) sh.mass[warp] = sum;
        __syncthreads();
        double cta = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) cta += sh.mass[w];
        const auto *got = tell(__double_as_longlong(cta), 0);
        double all = 0.0;
        for (int r = 0; r < a.ctas; ++r) all += __longlong_as_double(got[r][0]);
        return all;
    }

    // The cut, among the tokens that `inside` takes, of the first `k` of them (kCount), or
    // of the fewest first ones whose weights sum to `target`. lo <= the cut's logit <= hi.
    // kCount: where the first k fit into the list, top_p (below 1) is applied to them too,
    // and `both` is set. 0, which keeps everything, where there are fewer than k.
    template <bool kCount, typename F>
    __device__ unsigned long long find_cut(F inside, float lo, float hi, uint32_t k, double target, double top_p, bool &both) {
        double above = 0.0;   // mass and number of the tokens before hi
        uint32_t before = 0;
        both = false;
        for (bool first_turn = true;; first_turn = false) {
            // Bins of equal width, or by the bits of the logit where these are few: then
            // a bin is one value. lo and hi lie in different bins, so every turn narrows.
            const uint32_t k_hi = key_of(hi), range = k_hi - key_of(lo);
            const bool linear = range >= kBins && hi * 0.5f - lo * 0.5f > 1e-30f;
            const float scale = linear ? kBins / (hi * 0.5f - lo * 0.5f) : 0.0f;
            const int shift = max(0, 32 - __clz(range) - 10);
            static_assert(kBins == 1 << 10, "ten bits a turn");
            auto bin = [&](float x) -> int {
                return linear ? static_cast<int>(fminf((hi * 0.5f - x * 0.5f) * scale, kBins - 1.0f)) : static_cast<int>((k_hi - key_of(x)) >> shift);
            };
            for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
            if (threadIdx.x == 0) {
                sh.listed = 0;
                sh.star = kBins;
                sh.filled = 0;
            }
            __syncthreads();
            const int n = steps();
            for (int s = 0; s < n; ++s) {
                float v[E];
                load(s, v);
                const int i = index_of(s);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (v[e] >= lo && v[e] <= hi && inside(v[e], i + e)) atomicAdd(&sh.bins[bin(v[e])], 1u);
            }
            cluster_sync_all();
            // the row's counts, and sums of them and of about the weights up to each bin
            const int b = 2 * threadIdx.x;
            uint32_t c[2] = {0, 0};
            for (int r = 0; r < a.ctas; ++r) {
                const uint2 u = ld_cluster_u2(mapa_shared(smem_u32(&sh.bins[b]), r));
                c[0] += u.x;
                c[1] += u.y;
            }
            double about[2] = {0.0, 0.0};
            if constexpr (!kCount) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (c[j] != 0)
                        about[j] = c[j] * weight(linear ? fmaxf(lo, hi - (2 * (b + j) + 1) / scale) : value_of(k_hi - (static_cast<uint32_t>(b + j) << shift)));
            }
            double upto[2] = {static_cast<double>(c[0]) + c[1], about[0] + about[1]};
#pragma unroll
            for (int q = 0; q < (kCount ? 1 : 2); ++q) {
                upto[q] = warp_upto(upto[q], lane);
                if (lane == 31) sh.scan[q][warp] = upto[q];
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < (kCount ? 1 : 2); ++q)
                for (int w = 0; w < warp; ++w) upto[q] += sh.scan[q][w];
            const uint32_t up1 = static_cast<uint32_t>(upto[0]), up0 = up1 - c[1], up = up0 - c[0];  // tokens before b, up to b, up to b + 1
            // the bin in which the cut lies (kCount), or should lie
            const bool in1 = kCount ? before + static_cast<double>(up1) >= k : above + upto[1] >= target;
            const bool in0 = kCount ? before + static_cast<double>(up0) >= k : above + upto[1] - about[1] >= target;
            if (in0 || in1) atomicMin(&sh.star, in0 ? b : b + 1);
            if (c[0] + c[1] != 0) atomicMax(&sh.filled, c[1] != 0 ? b + 1 : b);
            __syncthreads();
            if (kCount && sh.star == kBins) return 0;
            const int star = min(sh.star, sh.filled);
            if (star / 2 == threadIdx.x) {
                sh.star_first = star & 1 ? up0 : up;
                sh.star_last = star & 1 ? up1 : up0;
                sh.from = sh.to = star;
            }
            __syncthreads();
            if constexpr (kCount) {
                both = first_turn && sh.star_last <= kList;
            } else {
                // and its neighbours, as far as the list holds them: the weights were estimated
                if (b <= star && sh.star_last - up <= kList / 2) atomicMin(&sh.from, b);
                else if (b + 1 <= star && sh.star_last - up0 <= kList / 2) atomicMin(&sh.from, b + 1);
                if (b + 1 >= star && up1 - sh.star_first <= kList / 2) atomicMax(&sh.to, b + 1);
                else if (b >= star && up0 - sh.star_first <= kList / 2) atomicMax(&sh.to, b);
                __syncthreads();
            }
            const int from = both ? 0 : sh.from, to = sh.to;
            if (from / 2 == threadIdx.x) sh.skipped = from & 1 ? up0 : up;
            if (to / 2 == threadIdx.x) sh.reached = to & 1 ? up1 : up0;
            if (threadIdx.x == kThreads - 1) sh.all = up1;
            __syncthreads();
            const uint32_t skipped = sh.skipped, reached = sh.reached, within = reached - skipped;
            const bool gather = within <= kList;
            // mass before these bins and in them; their tokens into the list; what bounds the three ranges
            double mass[2] = {0.0, 0.0};
            float low0 = INFINITY, low1 = INFINITY, high1 = -INFINITY, high2 = -INFINITY;
            const uint32_t listed0 = mapa_shared(smem_u32(&sh.listed), 0), list0 = mapa_shared(smem_u32(&sh.list[0]), 0);
            for (int s = 0; s < n; ++s) {
                float v[E];
                load(s, v);
                const int i = index_of(s);
                uint32_t in = 0, under = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!(v[e] >= lo && v[e] <= hi && inside(v[e], i + e))) continue;
                    const int at = bin(v[e]);
                    if (at < from) {
                        under |= 1u << e;
                        low0 = fminf(low0, v[e]);
                    } else if (at <= to) {
                        in |= 1u << e;
                        low1 = fminf(low1, v[e]);
                        high1 = fmaxf(high1, v[e]);
                        if (gather) {
                            const uint32_t place = add_cluster(listed0, 1u);
                            if (place < kList) st_cluster(list0 + place * 8, entry_of(v[e], i + e));
                        }
                    } else {
                        high2 = fmaxf(high2, v[e]);
                    }
                }
                if (!kCount && __any_sync(kAll, (in | under) != 0)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const double w = weight(v[e]);
                        mass[0] += under >> e & 1u ? w : 0.0;
                        mass[1] += in >> e & 1u ? w : 0.0;
                    }
                }
            }
            int range_of = 1;  // in which of the three the cut lies
            double sums[2] = {0.0, 0.0};
            if constexpr (!kCount) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    mass[q] = warp_sum(mass[q]);
                    if (lane == 0) sh.scan[q][warp] = mass[q];
                }
                __syncthreads();
                double cta[2] = {0.0, 0.0};
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    for (int w = 0; w < kWarps; ++w) cta[q] += sh.scan[q][w];
                const auto *got = tell(__double_as_longlong(cta[0]), __double_as_longlong(cta[1]));
                for (int r = 0; r < a.ctas; ++r) {
                    sums[0] += __longlong_as_double(got[r][0]);
                    sums[1] += __longlong_as_double(got[r][1]);
                }
                if (skipped > 0 && above + sums[0] >= target) range_of = 0;
                else if (above + (sums[0] + sums[1]) < target && sh.all > reached) range_of = 2;
            } else {
                cluster_sync_all();
            }
            if (range_of == 1 && gather) {
                if (rank == 0) finish<kCount>(within, both ? k : k - before - skipped, above + sums[0], target, both ? top_p : 1.0);
                cluster_sync_all();
                return sh.verdict;
            }
            if (range_of != 0) {
                above += sums[0] + (range_of == 2 ? sums[1] : 0.0);
                before += skipped;
            }
            auto outer = [](unsigned long long p, unsigned long long q) {
                return max(p >> 32, q >> 32) << 32 | max(p & 0xffffffffull, q & 0xffffffffull);
            };
            const float most = range_of == 0 ? hi : (range_of == 1 ? high1 : high2), least = range_of == 0 ? low0 : (range_of == 1 ? low1 : lo);
            const auto *got = tell(block_reduce(static_cast<unsigned long long>(key_of(most)) << 32 | (0xffffffffu - key_of(least)), 0, outer), 0);
            unsigned long long bounds = 0;
            for (int r = 0; r < a.ctas; ++r) bounds = outer(bounds, got[r][0]);
            hi = value_of(static_cast<uint32_t>(bounds >> 32));
            lo = value_of(0xffffffffu - static_cast<uint32_t>(bounds));
            if (lo >= hi) {
                const uint32_t equal = range_of == 1 ? within : (range_of == 0 ? skipped : sh.all - reached);
                uint32_t r = k - before;
                if constexpr (!kCount) {
                    const double w = weight(hi);
                    uint32_t short_of = 0;  // the least r that reaches the target, all of them where none does
                    r = equal;
                    while (r - short_of > 1) {
                        const uint32_t mid = short_of + (r - short_of) / 2;
                        if (above + mid * w >= target) r = mid;
                        else short_of = mid;
                    }
                }
                return entry_of(hi, nth_equal(hi, r, inside));
            }
        }
    }

    // Rank 0: the list sorted, summed and cut. want: how many of it (kCount).
    template <bool kCount>
    __device__ void finish(uint32_t n, uint32_t want, double above, double target, double top_p) {
        int size = 2;
        while (size < static_cast<int>(n)) size *= 2;
        for (int i = threadIdx.x; i < size; i += kThreads)
            if (i >= static_cast<int>(n)) sh.list[i] = 0;
        const int t = threadIdx.x;
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                __syncthreads();
                const int i = 2 * t - (t & (j - 1));
                if (i + j < size) {
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
            double w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = 2 * t + j;
                w[j] = i <= last ? weight(value_of(static_cast<uint32_t>(sh.list[i] >> 32))) : 0.0;
            }
            double upto = warp_upto(w[0] + w[1], lane), all = 0.0;
            if (lane == 31) sh.scan[0][warp] = upto;
            if (t == 0) sh.last = last;
            __syncthreads();
            for (int q = 0; q < kWarps; ++q) {
                if (q < warp) upto += sh.scan[0][q];
                all += sh.scan[0][q];
            }
            if (kCount) target = top_p * all;
            const double mid = above + (upto - w[1]);
            upto += above;
            if (2 * t <= last && mid >= target) atomicMin(&sh.last, 2 * t);
            else if (2 * t + 1 <= last && upto >= target) atomicMin(&sh.last, 2 * t + 1);
            __syncthreads();
            last = sh.last;
        }
        if (t < a.ctas) st_cluster(mapa_shared(smem_u32(&sh.verdict), t), sh.list[last]);
    }

    // The index of the r-th token (from 1) of logit x that `inside` takes, by rising index.
    template <typename F>
    __device__ int nth_equal(float x, uint32_t r, F inside) {
        const int n = steps();
        auto count = [&](int s) {
            float v[E];
            load(s, v);
            const int i = index_of(s);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c |= v[e] == x && inside(v[e], i + e) ? 1u << e : 0u;
            return c;
        };
        uint32_t mine = 0;
        for (int s = 0; s < n; ++s) mine += __popc(count(s));
        mine = __reduce_add_sync(kAll, mine);
        __syncthreads();
        if (lane == 0) sh.red[0][warp] = mine;
        __syncthreads();
        uint32_t cta = 0, before = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += static_cast<uint32_t>(sh.red[0][w]);
            cta += static_cast<uint32_t>(sh.red[0][w]);
        }
        const auto *got = tell(cta, 0);
        for (int q = 0; q < rank; ++q) before += static_cast<uint32_t>(got[q][0]);
        if (r > before && r <= before + mine) {
            uint32_t left = r - before;
            for (int s = 0; s < n; ++s) {
                const uint32_t c = count(s), k = __popc(c);
                uint32_t upto = k;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(kAll, upto, o);
                    if (lane >= o) upto += y;
                }
                const uint32_t all = __shfl_sync(kAll, upto, 31);
                if (left > all) {
                    left -= all;
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

template <typename T, bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) k_sample(SampleArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared sh;
    using R = Row<T, STAGED>;
    griddep_launch_dependents();
    const int64_t row = blockIdx.x / a.ctas;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    R r{a, sh, reinterpret_cast<T *>(dyn), x, static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)), static_cast<int>(blockIdx.x % a.ctas),
        static_cast<int>(threadIdx.x & 31), static_cast<int>(threadIdx.x >> 5)};
    griddep_wait();
    cluster_sync_all();  // every CTA of the row has started

    // the row into shared memory, its largest and least
    float best = -INFINITY, least = INFINITY;
    int best_at = -1;
    {
        const int n = r.steps();
        for (int s = 0; s < n; ++s) {
            alignas(16) T t[R::E];
            float v[R::E];
            r.fetch(s, t);
            if constexpr (STAGED) *reinterpret_cast<uint4 *>(r.staged(s)) = *reinterpret_cast<const uint4 *>(t);
            r.clean(t, v);
            const int i = r.index_of(s);
#pragma unroll
            for (int e = 0; e < R::E; ++e) {
                if (v[e] > best) {
                    best = v[e];
                    best_at = i + e;
                }
                if (v[e] > -INFINITY) least = fminf(least, v[e]);
            }
        }
    }
    {
        auto larger = [](unsigned long long p, unsigned long long q) { return max(p, q); };
        const unsigned long long top = r.block_reduce(best_at >= 0 ? entry_of(best, best_at) : 0ull, 0, larger);
        const unsigned long long low = r.block_reduce(0xffffffffu - key_of(least), 1, larger);
        const auto *got = r.tell(top, low);
        unsigned long long m = 0, l = 0;
        for (int q = 0; q < a.ctas; ++q) {
            m = max(m, got[q][0]);
            l = max(l, got[q][1]);
        }
        best_at = m != 0 ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(m)) : -1;
        best = m != 0 ? value_of(static_cast<uint32_t>(m >> 32)) : -INFINITY;
        least = value_of(0xffffffffu - static_cast<uint32_t>(l));
    }
    const float temperature = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    const int top_k = a.top_k != nullptr ? a.top_k[row] : 0;
    const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f, min_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    const float uniform = a.uniform[row];
    if (best_at < 0 || best == INFINITY || !(temperature > 0.0f) || top_k == 1 || top_p <= 0.0f) {
        if (r.rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = best_at;
            if (a.logprob != nullptr) a.logprob[row] = best_at < 0 ? NAN : 0.0f;
        }
        return;
    }
    r.weight = Weight{best, 1.4426950408889634074 / temperature};
    const Weight &weight = r.weight;
    least = fmaxf(least, static_cast<float>(fmax(best - 1000.0 / weight.per, -3.4e38)));  // below it weights are 0

    // the cut: kept are the tokens up to it in the order
    unsigned long long cut = 0;
    float cut_x = -INFINITY;
    int cut_i = 0x7fffffff;
    auto keep = [&](float v, int i) { return v > cut_x || (v == cut_x && i <= cut_i); };
    auto set_cut = [&](unsigned long long c) {
        if (c == 0) return;  // nothing is cut off
        cut = c;
        cut_x = value_of(static_cast<uint32_t>(c >> 32));
        cut_i = static_cast<int>(0xffffffffu - static_cast<uint32_t>(c));
    };
    bool done = false;
    if (top_k > 0 && top_k < a.vocab) {
        const unsigned long long c = r.template find_cut<true>(keep, least, best, static_cast<uint32_t>(top_k), 0.0, top_p < 1.0f ? static_cast<double>(top_p) : 1.0, done);
        set_cut(c);
    }
    if (top_p < 1.0f && !done) {
        const double sum = r.mass_of(keep);
        // The tokens lighter than (1 - top_p) of the mean weight weigh less than 1 - top_p together: the cut is above them.
        const double t = log2((1.0 - top_p) * sum / a.vocab) / weight.per;
        const double margin = 1e-6 * (fabs(static_cast<double>(best)) + fabs(t));
        const float lo = fmaxf(fmaxf(least, cut_x), static_cast<float>(fmax(best + t - margin, -3.4e38)));
        bool unused;
        set_cut(r.template find_cut<false>(keep, lo, best, 0u, static_cast<double>(top_p) * sum, 1.0, unused));
    }
    if (min_p > 0.0f) {
        // The least float whose weight is min_p or more: the logarithm's, or where that is
        // a step off (weights round to min_p over many floats: a largest logit near 0), by halving.
        const double at_least = min_p < 1.0f ? min_p : 1.0;
        uint32_t k = key_of(static_cast<float>(fmax(best + log2(at_least) / weight.per, -3.4e38)) + 0.0f);
        if (k > key_of(best) || weight(value_of(k)) < at_least || weight(value_of(k - 1)) >= at_least) {
            uint32_t under = key_of(-3.4e38f) - 1;
            k = key_of(best);
            while (k - under > 1) {
                const uint32_t mid = under + (k - under) / 2;
                if (weight(value_of(mid)) >= at_least) k = mid;
                else under = mid;
            }
        }
        const unsigned long long c = static_cast<unsigned long long>(k) << 32 | (0xffffffffu - 0x7fffffffu);
        if (c > cut) set_cut(c);
    }

    // the draw
    const double sum = r.mass_of(keep);
    const auto *parts = sh.slot[r.turn ^ 1];
    const double target = (uniform > 0.0f ? static_cast<double>(uniform) : 0.0) * sum;
    double before = 0.0;
    int owner = -1;
    for (int q = 0; q < a.ctas; ++q) {  // the first CTA that passes the target, else the last that holds anything
        const double m = __longlong_as_double(parts[q][0]);
        if (m > 0.0) {
            owner = q;
            if (before + m > target) break;
        }
        before += m;
    }
    if (owner != r.rank) return;
    before = 0.0;
    for (int q = 0; q < owner; ++q) before += __longlong_as_double(parts[q][0]);
    int owner_warp = -1;
    double at_warp = before;
    for (int w = 0; w < kWarps; ++w) {
        const double m = sh.mass[w];
        if (m > 0.0) {
            owner_warp = w;
            at_warp = before;
            if (before + m > target) break;
        }
        before += m;
    }
    if (owner_warp != r.warp) return;
    int found = -1;
    double found_w = 0.0;
    const int n = r.steps();
    for (int s = 0; s < n; ++s) {
        float v[R::E];
        double w[R::E], mine = 0.0;
        r.load(s, v);
        const int i = r.index_of(s);
#pragma unroll
        for (int e = 0; e < R::E; ++e) {
            w[e] = keep(v[e], i + e) ? weight(v[e]) : 0.0;
            mine += w[e];
        }
        const double upto = at_warp + warp_upto(mine, r.lane);
        const uint32_t passed = __ballot_sync(kAll, upto > target && mine > 0.0);
        const bool me = passed != 0 && r.lane == __ffs(passed) - 1;
        if (passed == 0 || me) {
            // this lane's token; where no lane passes, its last one so far
            double c = upto - mine;
#pragma unroll
            for (int e = 0; e < R::E; ++e) {
                if (w[e] > 0.0 && !(me && found >= i && c > target)) {
                    found = i + e;
                    found_w = w[e];
                    c += w[e];
                }
            }
        }
        if (passed != 0) {
            if (!me) found = -1;
            break;
        }
        at_warp = __shfl_sync(kAll, upto, 31);
    }
    const int token = __reduce_max_sync(kAll, found);
    if (found == token && token >= 0) {
        a.tokens[row] = token;
        if (a.logprob != nullptr) a.logprob[row] = static_cast<float>(log(found_w / sum));
    }
}

constexpr int kStageBytes = 96 * 1024;  // of a CTA: two share an SM

template <typename T, bool STAGED>
int launch_sample(const SampleArgs &a, int64_t rows, cudaStream_t st) {
    auto kern = k_sample<T, STAGED>;
    const int smem = STAGED ? a.slice * static_cast<int>(sizeof(T)) : 0;
    const int rc = ensure_max_smem(reinterpret_cast<const void *>(kern), kStageBytes, "sample");
    if (rc != LCML_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * a.ctas));
    cfg.blockDim = dim3(kThreads);
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
    // As few CTAs a row as hold it, then more while they find idle SMs.
    constexpr int kUnit = kWarps * Row<T, true>::kStep, E = Row<T, true>::E;
    const int64_t length = static_cast<int64_t>(a.vocab) + E - 1;
    auto slice = [&](int ctas) { return (length + static_cast<int64_t>(ctas) * kUnit - 1) / (static_cast<int64_t>(ctas) * kUnit) * kUnit; };
    a.ctas = 1;
    while (a.ctas < kMaxCluster && slice(a.ctas) * static_cast<int64_t>(sizeof(T)) > kStageBytes) a.ctas *= 2;
    while (a.ctas < kMaxCluster && rows * a.ctas * 2 <= sm_count() && slice(a.ctas) > kUnit) a.ctas *= 2;
    a.slice = static_cast<int>(slice(a.ctas));
    LCML_CHECK_ARG(rows * a.ctas <= 0x7fffffff, "lcml_sample: too many rows for one call");
    if (slice(a.ctas) * static_cast<int64_t>(sizeof(T)) > kStageBytes) return launch_sample<T, false>(a, rows, st);
    return launch_sample<T, true>(a, rows, st);
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
