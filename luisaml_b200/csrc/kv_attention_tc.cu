// Attention over the paged e4m3 cache: the tensor-core kernel for long runs of
// queries (prompts and chunks).
//
// One CTA per (sequence, cache head, 256 rows), rows = query * group + head as
// in kv_attention.cu, as two tiles of 128 rows that share every key and value
// tile of 128 tokens. Per tile t and key tile j:
//   S_t = sum over parts p of Q_t,p K_j^T    tcgen05 kind::f8f6f4, fp32 in TMEM
//   P_t = 2^(S_t scale + log2 s_v - m)       one thread per row, halves in TMEM over S_t
//   O_t += P_t V_j                           tcgen05 kind::f16, A from TMEM
// Keys go from global memory to the MMA as they are, against q's e4m3 parts
// (QScale, split_q). Two e4m3 products cost what one 16-bit product does, and
// no key is converted.
// Values are converted to halves (exact) by one warpgroup, from global memory
// into the MN-major 128-byte-swizzled layout of the B operand: the weights
// need more range than e4m3 has. They are rounded to halves, 2^-11 of each: A and
// B of the MMA have one type, and tf32 would halve its rate for the same 11 bits.
//
// Roles (16 warps): 0-3 and 4-7 softmax of tile 0 and 1 (a row per thread, no
// shuffles), 8-11 value conversion, 12 look-ups and TMA of the keys, 13 MMA
// issue. The MMA order PV_0(j) QK_0(j+1) PV_1(j) QK_1(j+1) lets one tile's
// softmax run under the other's products.
//
// With sinks (SINKS) the key tiles are those over the first positions, then the
// window's; a box of keys that no row sees is not looked up, its values are zeros.
// Masked tiles are weighed in one pass there. A unit of a short window is mostly set-up
// and end: of 42,700 clocks (window 512, 16 sinks, two row tiles of 32 + 8 heads of 128) 2,500
// look-ups and allocation, 9,000 q's load and split (12,000 with a division per row), 5,000
// the first tile's weights in two passes, 4,500 the output and the release.
//
// Bound: the tensor cores (4 head_dim FLOP per visible pair) and the
// exponentials, 16 a clock per SM: equal at head_dim 128, twice the products'
// time at 64. Measured at 128 (two prompts of up to 4096, 32 heads over 8, bf16):
// 225 us, 0.79 PFLOP/s (both of 4096: 318; with capped scores, which take every
// tile in the two passes of the masked ones, 613). A pair of key tiles takes 3450 clocks, of which the
// MMAs run 2048 and the weights of one row tile 1650. What was tried beside:
// P V of the first 64 keys under the weights of the others (one row tile 3360 ->
// 2860 clocks, two 3760 -> 3940), scores of 64 keys at a time (an MMA of half
// the keys takes as long: two 4050), two threads a row, CTAs that take over
// the units of others (235 and 241 us).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cstring>
#include <mutex>
#include <type_traits>

#include "lcml_attention.cuh"

namespace lcml {
namespace {

constexpr int kTile = 128;                // rows per tile, keys per tile
constexpr int kBlockRows = kTcBlockRows;  // rows per CTA: two tiles
static_assert(kBlockRows == 2 * kTile, "two tiles");
constexpr int kThreads = 512;
constexpr int kGroups = kTile / 16;       // 16-token groups of a key tile: one pair of scales each
constexpr int kInfoStages = 4;
constexpr int kVStages = 2;
// Of 8 pairs of weights, by polynomial (whole tiles): two prompts of 4096 take
// 328 us, 348 with none, 335 with 4 (head_dim 64: 269, 301, 293).
constexpr int kPolyPairs = 2;

// Registers per thread by role; 256 * 192 + 128 * 80 + 128 * 48 = 512 * 128,
// the block's allocation at launch.
constexpr int kSoftmaxRegs = 192, kConvertRegs = 80, kOtherRegs = 48;

struct alignas(16) GroupInfo {
    float k_scale, log2_v, inv_v;
    int row;  // cache row of the group's first token, -1: no token
};

template <int D, int NP>
struct Shape {
    static constexpr int kKStages = NP == 2 ? 3 : 2;
    static constexpr int kQPart = kTile * D;              // one part of one tile
    static constexpr int kQ = 2 * NP * kQPart;
    static constexpr int kK = kTile * D;                  // one stage
    static constexpr int kV = kTile * D * 2;              // one stage, halves
    static constexpr int kOffK = kQ;
    static constexpr int kOffV = kOffK + kKStages * kK;
    static constexpr int kSmem = kOffV + kVStages * kV + 1024;  // + alignment of the base
};

struct Shared {
    uint64_t k_full[3], k_empty[3], v_full[kVStages], v_empty[kVStages], info_full[kInfoStages], info_empty[kInfoStages];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int nan_seen;
    GroupInfo info[kInfoStages][kGroups];
    float row_factor[kBlockRows];
};

template <int N>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// D[tmem] (+)= A[tmem] * B[smem], halves -> f32.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors as {low, high} words. Only the start address (low
// 14 bits, in 16-byte units) changes between the steps of a tile, so a step is
// one 32-bit add.
__device__ __forceinline__ uint64_t desc_at(uint32_t low, uint32_t high) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
    return d;
}
// K-major operand of D-byte rows, D-byte swizzle (sdesc_kmajor<D>).
template <int D>
__device__ __forceinline__ uint32_t kmajor_low(uint32_t smem_addr) {
    return (smem_addr >> 4) | (1u << 16);
}
template <int D>
constexpr uint32_t kmajor_high() {
    return ((D == 128 ? 1024u : 512u) >> 4) | (1u << 14) | ((D == 128 ? 2u : 4u) << 29);
}
// B operand of P V: [token][d] with d contiguous (MN-major), halves, 128-byte
// swizzle: blocks of 64 d (128-byte rows, one per token, 8-token groups 1024
// bytes apart: the stride of K) of kTile tokens each (16 KiB apart: the stride
// of N).
__device__ __forceinline__ uint32_t values_low(uint32_t smem_addr) { return (smem_addr >> 4) | (((kTile * 128u) >> 4) << 16); }
constexpr uint32_t kValuesHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// kind::f16 with fp16 A and B, f32 D, A K-major, B MN-major.
constexpr uint32_t idesc_f16(uint32_t m, uint32_t n) { return (1u << 4) | (1u << 16) | ((n >> 3) << 17) | ((m >> 4) << 24); }

// Byte offset of 16-byte chunk `chunk` of row `row` in a K-major tile of
// D-byte rows with the D-byte swizzle (D = 128: chunk ^ row % 8, 64: chunk ^
// row / 2 % 4).
template <int D>
__device__ __forceinline__ uint32_t kmajor_offset(int row, int chunk) {
    return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

// a + b on two fp32 lanes.
__device__ __forceinline__ void add2(float &d0, float &d1, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\t"
        "mov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\t"
        "mov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// 2^x of two values on the FMA pipe, for part of a tile's weights: the special
// function unit alone takes 8 clocks a warp and value. n = round(x) by the
// addition of 1.5 * 2^23 (+ 127: the exponent field), 2^(x - n) by the
// degree-4 polynomial of least relative error on [-1/2, 1/2] (Remez exchange
// in 64 bits: 2.6e-6), far below the 2^-11 of the half it becomes. NaN stays NaN.
// A score may lie above its reference by any amount: x from 127 on gives 2^127,
// which the caller's limit on the weights refuses (unbounded, the exponent would
// run into the sign; a maximum of the arguments beside the weights spills: 251 us
// for two prompts of 4096, 242 with this).
__device__ __forceinline__ void exp2_poly(float &x0, float &x1) {
    constexpr float kMagic = 12582912.0f + 127.0f;
    auto clamp = [](float &x) {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-126.0f));
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(127.0f));
    };
    clamp(x0);
    clamp(x1);
    float t0, t1, f0, f1, p0, p1;
    add2(t0, t1, x0, x1, kMagic, kMagic);
    add2(f0, f1, t0, t1, -kMagic, -kMagic);
    fma2(f0, f1, f0, f1, -1.0f, -1.0f, x0, x1);
    fma2(p0, p1, f0, f1, 0.009570102207362652f, 0.009570102207362652f, 0.05591785907745361f, 0.05591785907745361f);
    fma2(p0, p1, p0, p1, f0, f1, 0.240247443318367f, 0.240247443318367f);
    fma2(p0, p1, p0, p1, f0, f1, 0.6931217908859253f, 0.6931217908859253f);
    fma2(p0, p1, p0, p1, f0, f1, 0.9999992847442627f, 0.9999992847442627f);
    mul2(x0, x1, p0, p1, __uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23));
}

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// Maximum and sum of 16 values as trees: one warp per scheduler and tile has
// to find its parallelism within the row.
__device__ __forceinline__ float max16(const uint32_t *r) {
    auto v = [&](int i) { return __uint_as_float(r[i]); };
    const float a = max3(v(0), v(1), v(2)), b = max3(v(3), v(4), v(5)), c = max3(v(6), v(7), v(8)), d = max3(v(9), v(10), v(11)),
                e = max3(v(12), v(13), v(14));
    return max3(max3(a, b, c), max3(d, e, v(15)), v(15));
}
__device__ __forceinline__ float sum16(const float *x) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 8; i += 2) add2(t[i], t[i + 1], x[i], x[i + 1], x[i + 8], x[i + 9]);
    add2(t[0], t[1], t[0], t[1], t[4], t[5]);
    add2(t[2], t[3], t[2], t[3], t[6], t[7]);
    add2(t[0], t[1], t[0], t[1], t[2], t[3]);
    return t[0] + t[1];
}

// Bits n .. 31.
__device__ __forceinline__ uint32_t bits_from(int n) { return n <= 0 ? 0xffffffffu : (n >= 32 ? 0u : 0xffffffffu << n); }

// The CTA's work, known to every thread.
template <bool SINKS>
struct Work {
    int seq, head, rows;      // rows in this block (<= kBlockRows)
    int row0;                 // first row within the sequence
    int t0, n, len, pos0;     // packed first token, queries, tokens held, position of query 0
    int lo, hi;               // the keys that some row sees (and the sinks)
    int tile_lo, tiles;       // first key tile of the window, and how many in all
    int sink_tiles;           // of which over the first keys, before the window's (SINKS)
    __device__ __forceinline__ int tile(int j) const { return SINKS && j < sink_tiles ? j : tile_lo + (SINKS ? j - sink_tiles : j); }
};

template <int D, int NP, bool CAP, bool SINKS>
__global__ void __launch_bounds__(kThreads, 1) k_kv_attention_tc(const __grid_constant__ CUtensorMap k_map, AttnArgs a, int box_rows,
                                                                 int min_rows) {
    using S = Shape<D, NP>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;

    griddep_launch_dependents();
    griddep_wait();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Units are handed out from the last one: within a sequence the last rows
    // see the most keys, and the longest units should not start last.
    Work<SINKS> w;
    const int sinks = SINKS ? a.sinks : 0;
    {
        w.head = blockIdx.x % a.c.kv_heads;
        const int64_t u = (gridDim.x - 1 - blockIdx.x) / a.c.kv_heads;
        w.seq = find_sequence(a.b.cu_tokens, a.b.batch, u, a.group, kBlockRows, 1);
        w.t0 = __ldg(a.b.cu_tokens + w.seq);
        const int t1 = static_cast<int>(min(static_cast<int64_t>(__ldg(a.b.cu_tokens + w.seq + 1)), a.b.total_tokens));
        const int held = __ldg(a.b.lengths + w.seq), len = max(0, held);
        w.n = w.t0 >= 0 ? max(0, t1 - w.t0) : 0;
        w.len = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(a.b.table_cols) * a.c.page_size));
        if ((w.len < len || held < 0 || w.n > a.max_tokens) && threadIdx.x == 0) record_device_error(a.err, kDevBadBatch);
        w.pos0 = w.len - w.n;
        const int64_t block = u - (static_cast<int64_t>(w.t0) * a.group / kBlockRows + w.seq);
        const int64_t all = static_cast<int64_t>(w.n) * a.group;
        // the whole CTA (block < 0: a unit before the first sequence's, where cu_tokens[0] > 0)
        if (block < 0 || block * kBlockRows >= all || all < min_rows || w.t0 < 0) return;
        w.row0 = static_cast<int>(block * kBlockRows);
        w.rows = static_cast<int>(min(static_cast<int64_t>(kBlockRows), all - w.row0));
        const int qa = w.row0 / a.group, qz = (w.row0 + w.rows - 1) / a.group;
        const int hi = a.causal ? min(w.pos0 + qz, w.len - 1) : w.len - 1;  // the last key any row sees
        const int lo = a.window > 0 ? max(0, w.pos0 + qa - a.window + 1) : 0;
        w.tile_lo = lo / kTile;
        w.sink_tiles = SINKS ? min((sinks + kTile - 1) / kTile, w.tile_lo) : 0;
        w.tiles = hi >= lo ? hi / kTile - w.tile_lo + 1 + w.sink_tiles : 0;
        w.lo = lo;
        w.hi = hi;
    }
    const bool two = w.rows > kTile;

    if (warp == 12) {
        if (lane == 0) {
            for (int i = 0; i < S::kKStages; ++i) {
                mbar_init(&sh.k_full[i], 1);
                mbar_init(&sh.k_empty[i], 1);
            }
            for (int i = 0; i < kVStages; ++i) {
                mbar_init(&sh.v_full[i], 4);
                mbar_init(&sh.v_empty[i], 1);
            }
            for (int i = 0; i < kInfoStages; ++i) {
                mbar_init(&sh.info_full[i], 1);
                mbar_init(&sh.info_empty[i], two ? 12 : 8);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.s_full[i], 1);
                mbar_init(&sh.q_full[i], 4);
                mbar_init(&sh.p_full[i], 4);
                mbar_init(&sh.o_full[i], 1);
            }
            sh.nan_seen = 0;
            fence_mbar_init();
        }
        tma_prefetch_desc(&k_map);
    }
    if (warp == 13) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int n = w.tiles;

    if (warp >= 12) {
        reg_dec<kOtherRegs>();
        if (warp == 12) {
            // Look-ups run two tiles ahead of their use: table entries for
            // j + 2 and scales for j + 1 are in flight while j is published.
            const int32_t *table = a.b.block_table + w.seq * a.b.table_stride;
            const int groups_per_box = box_rows / 16;
            // position of group `lane` of tile j, -1: no token (or, with sinks, in a box that no row sees)
            auto place = [&](int j) -> int64_t {
                const int64_t pos = static_cast<int64_t>(w.tile(j)) * kTile + lane * 16, box = pos - lane % groups_per_box * 16;
                return lane >= kGroups || j >= n || pos >= w.len || (SINKS && (box > w.hi || (box + box_rows <= w.lo && box >= sinks))) ? -1 : pos;
            };
            auto entry = [&](int j) -> int {  // page of group `lane` of tile j, -1: none
                const int64_t pos = place(j);
                return pos < 0 ? -1 : __ldg(table + pos / a.c.page_size);
            };
            auto row_of = [&](int j, int page) -> int {
                const int64_t pos = place(j);
                if (pos < 0) return -1;
                if (page < 0 || page >= a.c.num_pages) {
                    record_device_error(a.err, kDevBadPage);
                    return -1;
                }
                return static_cast<int>((static_cast<int64_t>(page) * a.c.kv_heads + w.head) * a.c.page_size + pos % a.c.page_size);
            };
            int row = row_of(0, entry(0));
            float ks = row >= 0 ? __ldg(a.c.k_scale + row / a.c.scale_block) : 0.0f, vs = row >= 0 ? __ldg(a.c.v_scale + row / a.c.scale_block) : 1.0f;
            int next_page = entry(1);
            int issued = 0;
            for (int j = 0; j < n; ++j) {
                const int later_page = entry(j + 2);
                const int next_row = row_of(j + 1, next_page);
                float next_ks = 0.0f, next_vs = 1.0f;
                if (next_row >= 0) {
                    next_ks = __ldg(a.c.k_scale + next_row / a.c.scale_block);
                    next_vs = __ldg(a.c.v_scale + next_row / a.c.scale_block);
                }
                const int st = j % kInfoStages;
                if (!__all_sync(0xffffffffu, mbar_wait(&sh.info_empty[st], ((j / kInfoStages) & 1) ^ 1, a.err, kDevTimeoutProducer))) break;
                if (lane < kGroups) {
                    const float sv = value_scale(vs);
                    sh.info[st][lane] = GroupInfo{row >= 0 ? ks : 0.0f, __log2f(sv), __fdividef(1.0f, sv), row};
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.info_full[st]);
                const int kst = j % S::kKStages;
                if (!__all_sync(0xffffffffu, mbar_wait(&sh.k_empty[kst], ((j / S::kKStages) & 1) ^ 1, a.err, kDevTimeoutProducer))) break;
                const bool lead = lane < kGroups && lane % groups_per_box == 0 && row >= 0;  // a box's first group has a token
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, lead));
                if (lane == 0) mbar_arrive_expect_tx(&sh.k_full[kst], boxes * box_rows * D);
                __syncwarp();
                if (lead)
                    asm volatile(
                        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                            smem + S::kOffK + kst * S::kK + lane * 16 * D),
                        "l"(&k_map), "r"(smem_u32(&sh.k_full[kst])), "r"(0), "r"(row)
                        : "memory");
                issued = j + 1;
                row = next_row;
                ks = next_ks;
                vs = next_vs;
                next_page = later_page;
            }
            // no copy is in flight when the CTA ends (only a given-up wait leaves any)
            for (int j = max(0, issued - S::kKStages); j < issued; ++j)
                mbar_wait(&sh.k_full[j % S::kKStages], (j / S::kKStages) & 1, a.err, kDevTimeoutDrain);
        } else if (warp == 13 && n > 0) {
            // The whole warp walks the schedule (uniform operands), one
            // elected lane issues: with a per-lane branch around the loop an
            // MMA takes 210 clocks to issue instead of the 64 it runs.
            constexpr uint32_t kIdescS = idesc_e4m3_f32(kTile, kTile, 0), kIdescO = idesc_f16(kTile, D);
            const bool lead = elect_one();
            auto wait = [&](uint64_t *bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, kDevTimeoutMma)) != 0; };
            auto qk = [&](int t, int j) {
                const uint32_t kb = kmajor_low<D>(smem + S::kOffK + (j % S::kKStages) * S::kK), qb = kmajor_low<D>(smem + t * NP * S::kQPart);
                if (lead) {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int k = 0; k < D / 32; ++k)
                            umma_f8f6f4(tmem + t * kTile, desc_at(qb + ((p * S::kQPart + k * 32) >> 4), kmajor_high<D>()),
                                        desc_at(kb + k * 2, kmajor_high<D>()), kIdescS, p + k > 0);
                    umma_commit(&sh.s_full[t]);
                }
            };
            bool ok = wait(&sh.k_full[0], 0) && wait(&sh.q_full[0], 0);
            if (ok) {
                qk(0, 0);
                if (two) {
                    ok = wait(&sh.q_full[1], 0);
                    if (ok) qk(1, 0);
                }
                if (lead) umma_commit(&sh.k_empty[0]);
            }
            for (int j = 0; j < n && ok; ++j) {
                const int vst = j % kVStages;
                const uint32_t vb = values_low(smem + S::kOffV + vst * S::kV);
                ok = wait(&sh.v_full[vst], (j / kVStages) & 1);
                for (int t = 0; t < (two ? 2 : 1) && ok; ++t) {
                    const bool last_tile = t == (two ? 1 : 0);
                    ok = wait(&sh.p_full[t], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            umma_f16_ts(tmem + 2 * kTile + t * D, tmem + t * kTile + k * 8, desc_at(vb + k * 128, kValuesHigh), kIdescO, k > 0 ? 1u : j > 0);
                        if (last_tile) umma_commit(&sh.v_empty[vst]);
                        if (j + 1 == n) umma_commit(&sh.o_full[t]);
                    }
                    if (j + 1 < n) {
                        const int kst = (j + 1) % S::kKStages;
                        if (t == 0) ok = wait(&sh.k_full[kst], ((j + 1) / S::kKStages) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        qk(t, j + 1);
                        if (last_tile && lead) umma_commit(&sh.k_empty[kst]);
                    }
                }
            }
        }
    } else if (warp >= 8) {
        reg_dec<kConvertRegs>();
        // A thread takes 16 codes of some tokens: global -> two 16-byte stores
        // of halves, the loads one tile ahead of the stores. Eight lanes take
        // four 16-code chunks (one 128-byte swizzled row of halves) of two
        // neighbouring tokens: their stores meet in no bank.
        constexpr int CH = D / 16;                 // 16-code chunks of a token
        constexpr int kPer = kTile * CH / 128;     // per thread and tile
        constexpr int kRowsPer = 128 / CH;         // tokens covered by the warpgroup at once
        const int wt = threadIdx.x - 256;
        const int ch = (wt & 3) + (D == 128 ? ((wt >> 3) & 1) * 4 : 0), tok0 = D == 128 ? ((wt >> 4) << 1) + ((wt >> 2) & 1) : wt >> 2;
        // keys that every row of the block sees: [all_lo, all_hi]
        const int qa = w.row0 / a.group, qz = (w.row0 + w.rows - 1) / a.group;
        const int all_hi = a.causal ? min(w.pos0 + qa, w.len - 1) : w.len - 1;
        const int all_lo = a.window > 0 ? max(0, w.pos0 + qz - a.window + 1) : 0;
        uint4 codes[kPer];
        auto fetch = [&](int j) -> bool {
            const int st = j % kInfoStages;
            if (!__all_sync(0xffffffffu, mbar_wait(&sh.info_full[st], (j / kInfoStages) & 1, a.err, kDevTimeoutProducer))) return false;
            const int64_t base = static_cast<int64_t>(w.tile(j)) * kTile;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int tok = tok0 + i * kRowsPer;
                const int row = sh.info[st][tok >> 4].row;
                codes[i] = make_uint4(0, 0, 0, 0);
                // with sinks: a slot that no row sees may hold NaN, which would cost a pass over the cache
                if (row >= 0 && base + tok < w.len && (!SINKS || (base + tok <= w.hi && (base + tok >= w.lo || base + tok < sinks))))
                    codes[i] = __ldg(reinterpret_cast<const uint4 *>(a.c.v + (static_cast<int64_t>(row) + (tok & 15)) * D) + ch);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.info_empty[st]);
            return true;
        };
        bool ok = n > 0 && fetch(0);
        for (int j = 0; j < n && ok; ++j) {
            const int vst = j % kVStages;
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.v_empty[vst], ((j / kVStages) & 1) ^ 1, a.err, kDevTimeoutProducer));
            if (!ok) break;
            const uint32_t vb = smem + S::kOffV + vst * S::kV;
            const int base = w.tile(j) * kTile;
            uint32_t nan = 0;
            if (base < all_lo || base + kTile - 1 > all_hi) {  // elsewhere a NaN reaches only rows that see it
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const uint32_t cw[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
                    for (int q = 0; q < 4; ++q) nan |= (cw[q] & 0x7f7f7f7fu) + 0x01010101u;
                }
            }
            if (__any_sync(0xffffffffu, (nan & 0x80808080u) != 0)) {
                // NaN codes: zeros here, so 0 * NaN reaches no row that does
                // not see them; the rows that do get theirs at the end
                sh.nan_seen = 1;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    uint32_t *cw = reinterpret_cast<uint32_t *>(&codes[i]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) cw[q] &= ~(((((cw[q] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu);
                }
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int tok = tok0 + i * kRowsPer;
                const uint32_t cw[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
                uint32_t h[8];
#pragma unroll
                for (int q = 0; q < 4; ++q) e4m3x4_to_half2(cw[q], h[2 * q], h[2 * q + 1]);
                const uint32_t row = vb + (ch >> 2) * (kTile * 128) + tok * 128;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t at = row + ((((ch & 3) * 2 + half) ^ (tok & 7)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(h[4 * half]), "r"(h[4 * half + 1]), "r"(h[4 * half + 2]),
                                 "r"(h[4 * half + 3])
                                 : "memory");
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[vst]);
            if (j + 1 < n) ok = fetch(j + 1);
        }
    } else {
        reg_inc<kSoftmaxRegs>();
        const int t = warp >> 2;
        if (t == 0 || two) {
            // Q tile -> e4m3 parts. A lane takes 8 elements of a row: 16 lanes
            // a row at head_dim 128, 8 at 64; a warp its tile's rows
            // warp % 4 * 32 .. + 31. Rows past the block's end are zeros.
            {
                constexpr int LPR = D / 8, RPW = 32 / LPR, kPasses = 32 / RPW;
                const int part_lane = lane % LPR, r0 = warp * 32 + lane / LPR;
                const bool vec = aligned(a.q, 16) && a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
                uint4 e8[kPasses];  // all loads at once: one latency
                uint32_t mx[kPasses];
                // the pass's row, RPW rows on each time: one division in all
                int in_group = (w.row0 + r0) % a.group;
                const int more_queries = RPW / a.group, more_heads = RPW % a.group;
                const uint16_t *p = static_cast<const uint16_t *>(a.q) + (w.t0 + static_cast<int64_t>((w.row0 + r0) / a.group)) * a.q_token_stride +
                                    (static_cast<int64_t>(w.head) * a.group + in_group) * a.q_head_stride + part_lane * 8;
                const int64_t step = more_queries * a.q_token_stride + more_heads * a.q_head_stride, wrap = a.q_token_stride - a.group * a.q_head_stride;
#pragma unroll
                for (int u = 0; u < kPasses; ++u) {
                    const int r = r0 + u * RPW;
                    e8[u] = make_uint4(0, 0, 0, 0);
                    if (r < w.rows) {
                        if (vec) {
                            e8[u] = __ldg(reinterpret_cast<const uint4 *>(p));
                        } else {
                            uint32_t h[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) h[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
                            e8[u] = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                    p += step;
                    in_group += more_heads;
                    if (in_group >= a.group) {
                        in_group -= a.group;
                        p += wrap;
                    }
                }
                // a row's largest magnitude: 16-bit floats order like their bits (NaN above infinity)
#pragma unroll
                for (int u = 0; u < kPasses; ++u) {
                    const uint32_t h[4] = {e8[u].x & 0x7fff7fffu, e8[u].y & 0x7fff7fffu, e8[u].z & 0x7fff7fffu, e8[u].w & 0x7fff7fffu};
                    const uint32_t m2 = __vmaxu2(__vmaxu2(h[0], h[1]), __vmaxu2(h[2], h[3]));
                    mx[u] = max(m2 & 0xffffu, m2 >> 16);
                }
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int u = 0; u < kPasses; ++u) mx[u] = max(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], o));
#pragma unroll
                for (int u = 0; u < kPasses; ++u) {
                    const int r = r0 + u * RPW;
                    const uint32_t h[4] = {e8[u].x, e8[u].y, e8[u].z, e8[u].w};
                    const QScale<NP> qs(mx[u]);
                    if (part_lane == 0) sh.row_factor[r] = qs.factor;
                    uint32_t lo[NP], hi[NP];
                    split_q<NP>(h[0], h[1], qs, lo);
                    split_q<NP>(h[2], h[3], qs, hi);
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        const uint32_t at = smem + (t * NP + p) * S::kQPart + kmajor_offset<D>(r & 127, part_lane >> 1) + (part_lane & 1) * 8;
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(lo[p]), "r"(hi[p]) : "memory");
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full[t]);
            }
            const int r = threadIdx.x;  // row of the block
            const int row = w.row0 + r;
            const bool live = r < w.rows;  // the others (zero queries) are computed and dropped
            const int pos = w.pos0 + row / a.group;
            const int last = a.causal ? min(pos, w.len - 1) : w.len - 1;
            const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            const float factor = sh.row_factor[r] * (CAP ? a.inv_cap : a.scale_log2);  // this warp's own rows
            const uint32_t lane_base = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lanes 32 (warp % 4) ..
            const uint32_t ts = tmem + lane_base + t * kTile, to = tmem + lane_base + 2 * kTile + t * D;
            // which of 32 keys from k0 on the row sees
            auto row_sees = [&](int k0) { return (bits_from(first - k0) | ~bits_from(sinks - k0)) & ~bits_from(last + 1 - k0); };
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const int st = j % kInfoStages;
                ok = mbar_wait(&sh.info_full[st], (j / kInfoStages) & 1, a.err, kDevTimeoutEpilogue) &&
                     mbar_wait(&sh.s_full[t], j & 1, a.err, kDevTimeoutEpilogue);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const int base = w.tile(j) * kTile;
                const bool plain = !CAP && __all_sync(0xffffffffu, (first <= base || (SINKS && base + kTile <= sinks)) && last >= base + kTile - 1);
                const GroupInfo *info = sh.info[st];
                uint32_t sr[2][32], p[64];
                // Weights of the tile against the reference maximum, 32 scores
                // at a time and the next 32 on their way. Returns the largest
                // sum of 16 weights, a bound of each. kRaw: S as the MMA left
                // it, else in log2 units.
                // kMasked: with the row's mask.
                auto weights = [&](auto raw, auto masked, float ref, float &sum) {
                    constexpr bool kRaw = decltype(raw)::value, kMasked = decltype(masked)::value;
                    float most = 0.0f;
                    tmem_ld_32x32b_x32(ts, sr[0]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 g0 = *reinterpret_cast<const float4 *>(info + 2 * q), g1 = *reinterpret_cast<const float4 *>(info + 2 * q + 1);
                        tmem_wait_ld();
                        if (q < 3) tmem_ld_32x32b_x32(ts + (q + 1) * 32, sr[(q + 1) & 1]);
                        // keys of these 32 that the row sees
                        uint32_t seen = 0;
                        if constexpr (kMasked) {
                            seen = row_sees(base + q * 32);
                            if (!__any_sync(0xffffffffu, seen != 0)) {  // of no row of the warp
#pragma unroll
                                for (int e = 0; e < 16; ++e) p[q * 16 + e] = 0;
                                continue;
                            }
                        }
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float f = kRaw ? (g ? g1.x : g0.x) * factor : 1.0f, b = (kRaw ? (g ? g1.y : g0.y) : 0.0f) - ref;
                            float x[16];
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                fma2(x[e], x[e + 1], __uint_as_float(sr[q & 1][g * 16 + e]), __uint_as_float(sr[q & 1][g * 16 + e + 1]), f, f, b, b);
                                if constexpr (kMasked) {
                                    x[e] = seen >> (g * 16 + e) & 1u ? x[e] : -INFINITY;
                                    x[e + 1] = seen >> (g * 16 + e + 1) & 1u ? x[e + 1] : -INFINITY;
                                }
                                if (kRaw && !kMasked && e / 2 < kPolyPairs) {
                                    exp2_poly(x[e], x[e + 1]);
                                } else {
                                    x[e] = exp2_approx(x[e]);
                                    x[e + 1] = exp2_approx(x[e + 1]);
                                }
                                const __half2 hp = __floats2half2_rn(x[e], x[e + 1]);
                                p[q * 16 + g * 8 + e / 2] = *reinterpret_cast<const uint32_t *>(&hp);
                            }
                            const float of16 = sum16(x);
                            most = fmaxf(most, of16);
                            sum = fmaf(of16, g ? g1.z : g0.z, sum);
                        }
                    }
                    return most;
                };
                // The reference maximum moves only when a weight passes 2^8 (a
                // half has room for that), so after the first tile the weights
                // are taken against the old one at once, without a pass for
                // the maximum; a tile with 16 weights of a larger sum (in any
                // row of the warp) is done again below. S stays until P is
                // known to be good.
                bool done = false;
                if ((plain || (SINKS && !CAP)) && __all_sync(0xffffffffu, m > -INFINITY)) {
                    float sum = l, most;
                    if constexpr (SINKS && !CAP) {
                        // Most tiles of a short window are masked: of two prompts of 4096 with a window of 512 and 16
                        // sinks this saves 11 of 180 us against the two passes below, of chunks of 1000 6 of 83.
                        if (plain) most = weights(std::true_type{}, std::false_type{}, m, sum);
                        else most = weights(std::true_type{}, std::true_type{}, m, sum);
                    } else {
                        most = weights(std::true_type{}, std::false_type{}, m, sum);
                    }
                    done = !__any_sync(0xffffffffu, most > 256.0f);
                    if (done) l = sum;
                }
                if (!done) {
                    // scores in log2 units, masked, in place of S; their maximum
                    float top = -INFINITY;
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        uint32_t(&r)[32] = sr[0];
                        if constexpr (SINKS) {
                            if (!__any_sync(0xffffffffu, row_sees(base + q * 32) != 0)) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(-INFINITY);
                                tmem_st_32x32b_x32(ts + q * 32, r);
                                continue;
                            }
                        }
                        tmem_ld_32x32b_x32(ts + q * 32, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float2 gi = *reinterpret_cast<const float2 *>(info + 2 * q + (e >> 4));
                            const int k = base + q * 32 + e;
                            const float x = __uint_as_float(r[e]), f = gi.x * factor;
                            const float y = CAP ? cap_score(x, f, a.cap) + gi.y : fmaf(x, f, gi.y);
                            r[e] = __float_as_uint((k >= first || (SINKS && k < sinks)) && k <= last ? y : -INFINITY);
                        }
                        top = max3(top, max16(r), max16(r + 16));
                        tmem_st_32x32b_x32(ts + q * 32, r);
                    }
                    tmem_wait_st();
                    // The S of this tile being full means that the previous P V is done.
                    if (__any_sync(0xffffffffu, top > m + (plain ? 0.0f : 8.0f))) {
                        const float nm = fmaxf(m, top);
                        const float f = nm == m ? 1.0f : exp2_approx(m - nm);
                        m = nm;
                        l *= f;
                        if (j > 0) {
#pragma unroll 1
                            for (int q = 0; q < D / 32; ++q) {
                                uint32_t(&o)[32] = sr[0];
                                tmem_ld_32x32b_x32(to + q * 32, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st_32x32b_x32(to + q * 32, o);
                            }
                        }
                    }
                    weights(std::false_type{}, std::false_type{}, m == -INFINITY ? 0.0f : m, l);
                }
                tmem_st_32x32b_x32(ts, reinterpret_cast<uint32_t(&)[32]>(p[0]));
                tmem_st_32x32b_x32(ts + 32, reinterpret_cast<uint32_t(&)[32]>(p[32]));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sh.p_full[t]);
                    mbar_arrive(&sh.info_empty[st]);
                }
            }
            if (ok && n > 0) ok = mbar_wait(&sh.o_full[t], 0, a.err, kDevTimeoutEpilogue);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            // one row per thread, in whole 32-byte sectors where aligned
            const int64_t token = w.t0 + static_cast<int64_t>(row / a.group);
            const int qh = w.head * a.group + row % a.group;
            uint16_t *out = static_cast<uint16_t *>(a.out) + token * a.out_token_stride + qh * a.out_head_stride;
            const bool vec = aligned(a.out, 32) && a.out_token_stride % 16 == 0 && a.out_head_stride % 16 == 0;
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
                uint32_t o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0;
                if (ok && n > 0) {
                    tmem_ld_32x32b_x32(to + q * 32, o);
                    tmem_wait_ld();
                }
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float y0 = l != 0.0f ? __uint_as_float(o[2 * e]) * inv : 0.0f, y1 = l != 0.0f ? __uint_as_float(o[2 * e + 1]) * inv : 0.0f;
                    if (NP == 2) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(y0, y1);
                        pk[e] = *reinterpret_cast<const uint32_t *>(&b);
                    } else {
                        const __half2 b = __floats2half2_rn(y0, y1);
                        pk[e] = *reinterpret_cast<const uint32_t *>(&b);
                    }
                }
                if (vec && live && ok) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + q * 32 + e * 16), "r"(pk[8 * e]),
                                     "r"(pk[8 * e + 1]), "r"(pk[8 * e + 2]), "r"(pk[8 * e + 3]), "r"(pk[8 * e + 4]), "r"(pk[8 * e + 5]),
                                     "r"(pk[8 * e + 6]), "r"(pk[8 * e + 7])
                                     : "memory");
                } else if (live && ok) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        out[q * 32 + 2 * e] = static_cast<uint16_t>(pk[e]);
                        out[q * 32 + 2 * e + 1] = static_cast<uint16_t>(pk[e] >> 16);
                    }
                }
                __syncwarp();
            }
            if (live && ok && a.lse != nullptr)
                a.lse[token * (static_cast<int64_t>(a.c.kv_heads) * a.group) + qh] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 13) tmem_dealloc(tmem, 512);

    // Values with NaN codes were met (and counted as zeros): give the rows
    // that see them their NaN, column by column, from the cache itself.
    if (sh.nan_seen && static_cast<int>(threadIdx.x) < w.rows) {
        const int row = w.row0 + threadIdx.x;
        const int pos = w.pos0 + row / a.group;
        const int last = a.causal ? min(pos, w.len - 1) : w.len - 1, first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        const int32_t *table = a.b.block_table + w.seq * a.b.table_stride;
        uint16_t *out = static_cast<uint16_t *>(a.out) + (w.t0 + static_cast<int64_t>(row / a.group)) * a.out_token_stride +
                        (w.head * a.group + row % a.group) * a.out_head_stride;
        for (int k = min(first, sinks) > 0 ? 0 : first; k <= last; ++k) {
            if (SINKS && k == sinks && k < first) k = first;
            const int64_t page = __ldg(table + k / a.c.page_size);
            if (page < 0 || page >= a.c.num_pages) continue;
            const uint32_t *v = reinterpret_cast<const uint32_t *>(a.c.v + ((page * a.c.kv_heads + w.head) * a.c.page_size + k % a.c.page_size) * D);
            for (int i = 0; i < D / 4; ++i) {
                const uint32_t bad = ((__ldg(v + i) & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                if (bad != 0)
                    for (int b = 0; b < 4; ++b)
                        if (bad >> (8 * b + 7) & 1u) out[i * 4 + b] = 0x7fff;  // NaN in both types
            }
        }
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// Key boxes: the largest power of two of tokens that divides a page and a
// tile, so no box crosses a page.
int box_rows_of(const lcml_kv_cache *c) {
    int r = 16;
    while (r < kTile && c->page_size % (2 * r) == 0) r *= 2;
    return r;
}

template <int D, int NP, bool CAP>
int launch_tc(const lcml_kv_attention_desc *d, const AttnArgs &a, int min_rows, cudaStream_t st) {
    using S = Shape<D, NP>;
    auto fn = encode_fn();
    if (!fn) return set_error(LCML_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    CUtensorMap map;
    memset(&map, 0, sizeof(map));
    const int box = box_rows_of(d->cache);
    cuuint64_t dims[2] = {D, static_cast<cuuint64_t>(d->cache->num_pages) * d->cache->kv_heads * d->cache->page_size};
    cuuint64_t strides[1] = {D};
    cuuint32_t bx[2] = {D, static_cast<cuuint32_t>(box)};
    cuuint32_t es[2] = {1, 1};
    const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, d->cache->k, dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(LCML_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    // a kernel without the sinks' tests: they cost two prompts of 4096, which have none, 8 us of 232
    auto kern = a.sinks > 0 ? k_kv_attention_tc<D, NP, CAP, true> : k_kv_attention_tc<D, NP, CAP, false>;
    const int rc = ensure_max_smem(reinterpret_cast<const void *>(kern), S::kSmem, "kv_attention_tc");
    if (rc != LCML_OK) return rc;
    const int64_t units = (d->batch->total_tokens * a.group / kBlockRows + d->batch->batch) * d->cache->kv_heads;
    LCML_CHECK_ARG(units <= 0x7fffffff, "lcml_kv_attention: too much work for one call");
    return launch_dependent(kern, dim3(static_cast<unsigned>(units)), kThreads, S::kSmem, st, "kv_attention_tc", map, a, box, min_rows);
}

template <int D>
int dispatch_tc(const lcml_kv_attention_desc *d, const AttnArgs &a, int min_rows, cudaStream_t st) {
    if (a.bf16) return a.cap != 0.0f ? launch_tc<D, 2, true>(d, a, min_rows, st) : launch_tc<D, 2, false>(d, a, min_rows, st);
    return a.cap != 0.0f ? launch_tc<D, 3, true>(d, a, min_rows, st) : launch_tc<D, 3, false>(d, a, min_rows, st);
}

}// namespace

// Cache rows are 32-bit TMA coordinates; a negative softmax_scale would turn
// the maximum of a group into its minimum.
bool kv_attention_tc_fits(const lcml_kv_attention_desc *d) {
    const lcml_kv_cache *c = d->cache;
    return (c->head_dim == 64 || c->head_dim == 128) && d->softmax_scale >= 0.0f && c->num_pages > 0 &&
           c->num_pages * c->kv_heads * c->page_size <= 0x7fffffff;
}

int kv_attention_tc(const lcml_kv_attention_desc *d, const AttnArgs &a, int min_rows, cudaStream_t st) {
    return d->cache->head_dim == 64 ? dispatch_tc<64>(d, a, min_rows, st) : dispatch_tc<128>(d, a, min_rows, st);
}

}// namespace lcml
