// Attention over the paged e4m3 cache: the streaming kernel (decode steps and
// short runs of queries) and the entry points.
//
// Rows of a sequence and cache head are its n queries x group heads, r = query
// * group + head, in tiles of 8 or 16. A segment is one row tile of one cache
// head over all the keys it sees, in steps of 16 keys. The batch's segments
// lie end to end in one list of steps, and every CTA of a grid that fits the
// machine once takes an equal stretch of it, whatever the lengths: no CTA is
// idle and none is late. Within a CTA warp w takes steps w, w + kWarps, ...;
// its ring of copies runs on over segment ends.
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T, with
// keys and d on the 16-row side of mma.m16n8k16 and 8 query rows on the other:
// a decode step's 8 rows fill the tile (as the 16-row side they would leave
// half of it, and half of the accumulators, empty). Keys and values go from
// global memory through the per-lane cp.async ring straight into the fragment
// layout: the dot product's order of d is free, so a lane's key fragments are
// 16 consecutive bytes of two key rows, and O^T's row is free too, so a lane
// reads consecutive bytes of four value rows and pairs them by byte permutes.
// Every lane reads back only what it copied itself: no barriers, no bank
// conflicts. Codes become halves by one exact conversion per pair (mma.sync
// takes e4m3 operands too, but converts them itself for every use: measured
// slower); the block scales multiply the scores (keys) and join the exponent
// (values, value_scale()). P^T reaches its operand layout by one movmatrix per
// 8 keys. The weights are rounded to halves for their product, 2^-11 of each: codes
// are exact in halves and both operands of the MMA have one type; in tf32 (the
// same 11 bits) the product would take twice the instructions. Sums keep fp32.
//
// At a segment's end each warp leaves its (m, l, O) in shared memory and goes
// on; the last of them joins and writes. A segment that lies in several CTAs
// leaves (m, l, O) per CTA, which k_kv_attention_join merges in list order
// (deterministic: the warps' shares are joined in warp order by whichever comes
// last). Where no sequence can be longer than kWholeSteps, a CTA takes whole
// segments and there is nothing to join.
//
// Bound: HBM, 2 head_dim bytes per key and cache head (one token of a
// 131072-token sequence, 8 cache heads of 128: 65 us, 4.2 of a copy's 6.5 TB/s:
// 5.3 TB/s while it streams, the rest is the plan, the first copies and the
// join; of 64 sequences of up to 4096: 77 us). Several tokens at head_dim 256 have
// no other kernel than this one's tiles of 8 rows, which copy and convert the keys
// once per tile: 4 tokens of 16 sequences of 2000 66 us (floor 20), a prompt of
// 4096 5.6 ms (floor 166 us).
#include "lcml_attention.cuh"

namespace lcml {
namespace {

constexpr int kStep = 16;          // keys per warp step
// Up to here segments are not split. With many of them that is faster: 32 steps
// in one CTA or split, one token of 64 sequences of 500 25.9 and 27.2 us
// (head_dim 64: 14.7 and 19.2). With few it is not, 12.1 and 11.0 for 1
// sequence: the number of segments, which the host can bound, is not looked at yet.
constexpr int kWholeSteps = 64;
constexpr int kMaxBatch = 1024;    // sequences per launch (the plan's table in shared memory)

// Which kernel: the streaming one takes 1.0 us of an SM for 16 rows and 128
// keys (0.7 at head_dim 64), the tensor-core one 1.9 us for up to 256 rows, but
// it splits no keys: with fewer units than SMs the rest of the machine idles.
// Both are proportional to the keys, so the lengths, which the host does not
// know, cancel out: the tensor-core kernel wins from `rows` rows a unit or SM,
// whichever are more. 8 cache heads, streaming / tensor-core in us:
//   head_dim 128, 64 sequences of 4096: 16 rows 135 / 249, 32 250 / 256, 64 484 / 256
//     8 sequences of 32768: 32 rows 228 / 420, 64 433 / 420, 96 634 / 445
//     1 sequence of 32768: 256 rows 204 / 497, 512 392 / 500
//   head_dim 64, 64 of 4096: 32 rows 169 / 217, 64 318 / 219
//     8 of 32768: 64 rows 274 / 380, 96 404 / 380
constexpr int tc_rows(int head_dim) { return head_dim == 64 ? 40 : 28; }

// Warps per CTA and CTAs per SM: 8 warps an SM with deep rings of copies (16 at
// head_dim 64). Two CTAs of four, so that one's set-up and join run under the
// other's copies: one token of 200 sequences of 500, 8 cache heads, 85 us with
// one CTA of eight, 64 here; of 64 x 500 34 and 26, of 64 x 4096 118 and 119, of
// 8 x 300 10.9 and 12.7. Four CTAs of two: 59, 23, 121 and 14.7, but 14.8 for
// one sequence of 500 (11.4 and 12.1). 16-row tiles at head_dim 64 keep two CTAs
// of eight: their shares of O leave no room for four of four (4 tokens of 64
// sequences of 1000: 41 and 57 us).
constexpr int stream_warps(int head_dim, int groups) { return head_dim == 64 && groups == 2 ? 8 : 4; }
constexpr int stream_ctas(int head_dim, int groups) { return head_dim == 64 && groups == 1 ? 4 : 2; }

template <int D, int RG>
struct Shape {
    static constexpr int kWarps = stream_warps(D, RG);
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = 8 * RG;                           // rows per tile
    static constexpr int kCtasPerSm = stream_ctas(D, RG);
    // Steps a CTA takes at least (one token of one sequence of 1000: 10.6 us,
    // 11.4 with twice as many, 13.7 with four times), and what a segment's set-up
    // and join cost in steps (of one sequence of 2000 11.7 us, 13.9 with none;
    // of 200 sequences of 500 64.9, 63.5 with none, 67.3 with half as much again).
    // 16-row tiles join twice as much: 4 tokens of 16 sequences of up to 2000, head_dim
    // 64, 28.0 us, 29.7 with 2 kWarps (64 x 1000 at 128: 52.7 and 51.7).
    static constexpr int kMinRange = 2 * kWarps, kPad = (RG == 1 ? 2 : 3) * kWarps;
    static constexpr int kStages = D == 256 ? 2 : 4;
    static constexpr int kStageBytes = 2 * kStep * D;              // per warp
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kShare = kRows * D;                       // floats of one warp's O
    static constexpr int kJoin = kWarps * kShare * 4;
    static constexpr int kPlan = kMaxBatch * 12 + 16;              // first step and steps per segment of each sequence
    static constexpr int kSmem = kRing + kJoin + kPlan;
};

// Where 16-byte chunk q of row r of a warp's share lies: rows of D floats, the
// chunks of each 128 bytes permuted so that neither the fragment-order stores
// (8 lanes: four rows 2c + e, two runs of d) nor the row-order loads (8
// consecutive chunks) meet in a bank.
template <int D>
__device__ __forceinline__ int share_chunk(int r, int q) {
    const int line = q >> 3, c = (r >> 1) & 3;
    const int turn = D == 64 ? (c & 1) | (c >> 1) << 2 : (D == 128 ? c : c | (line & 1) << 2);
    return r * (D / 4) + line * 8 + ((q & 7) ^ turn);
}

// A segment cut by CTA boundaries: CTAs first .. first + pieces - 1 hold its pieces.
struct JoinItem {
    int pieces, rows;
    int row0, t0;  // the tile's first row within the sequence, the sequence's first packed token
    int head;
    int pad[3];
};

struct Span {
    int n, len, lo, steps, tiles;
    int t0;    // first packed token
    int pos0;  // position of query 0 (negative: queries before the first token see nothing)
    bool cut;  // longer than the call's bounds, or of negative length
};

// Sequence s; steps counts from lo over all the keys any of its queries sees,
// and PAD empty ones: CTAs with many short segments would be late otherwise
// (and a row without keys still gets its zeros).
template <int ROWS, int PAD>
__device__ __forceinline__ Span span_of(const AttnArgs &a, int s) {
    Span r;
    r.t0 = __ldg(a.b.cu_tokens + s);
    const int t1 = static_cast<int>(min(static_cast<int64_t>(__ldg(a.b.cu_tokens + s + 1)), a.b.total_tokens));
    const int held = __ldg(a.b.lengths + s);
    const int n = r.t0 >= 0 ? max(0, t1 - r.t0) : 0, len = max(0, held);
    r.n = static_cast<int>(min(static_cast<int64_t>(n), a.max_tokens));
    r.len = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(a.b.table_cols) * a.c.page_size));
    r.cut = r.n < n || r.len < len || held < 0;
    r.pos0 = r.len - n;
    const int64_t first = static_cast<int64_t>(r.pos0) - a.window + 1;  // the first query's oldest key
    r.lo = a.window > 0 && first > 0 ? static_cast<int>(first) & ~(kStep - 1) : 0;
    r.steps = (r.len - r.lo + kStep - 1) / kStep + PAD;
    r.tiles = static_cast<int>((static_cast<int64_t>(r.n) * a.group + ROWS - 1) / ROWS);
    return r;
}

template <int BYTES>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void *src, uint32_t bytes) {
    if constexpr (BYTES == 16) cp_async_16_zfill(dst, src, bytes);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

// D += A (16x16, row) * B (16x8, col), halves, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transpose of an 8x8 matrix of halves held as fragments (lane: row g, columns 2c, 2c + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Bounded wait of a warp until another has set *flag (shared memory) to `value`.
__device__ __forceinline__ bool wait_for(const int *flag, int value, int *err) {
    const volatile int *f = flag;
    bool ok = true;
    if (*f != value) {
        const long long t0 = clock64();
        while (*f != value && ok) ok = clock64() - t0 <= kWaitLimitCycles;
        if (!ok) record_device_error(err, kDevTimeoutEpilogue);
    }
    ok = __all_sync(0xffffffffu, ok);
    __threadfence_block();
    return ok;
}

// Bytes of w that hold a NaN code (0x7f or 0xff), as the e4m3 code of 1.0 there and 0 elsewhere.
__device__ __forceinline__ uint32_t nan_ones(uint32_t w) {
    const uint32_t m = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bit 7 of each NaN byte
    return (m >> 7) * 0x38u;
}
__device__ __forceinline__ uint32_t nan_cleared(uint32_t w) {
    const uint32_t m = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~((m >> 7) * 0xffu);
}

template <int D, int RG, bool BF16, bool CAP>
__global__ void __launch_bounds__(Shape<D, RG>::kThreads, Shape<D, RG>::kCtasPerSm) k_kv_attention(AttnArgs a, int max_rows, bool whole, int part_rows,
                                                                                          JoinItem *join_items, float *part_ml, float *part_o) {
    using S = Shape<D, RG>;
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kStages = S::kStages, kRows = S::kRows;
    constexpr int KC = D / 64;        // 16-byte pieces of a key row per lane
    constexpr int VB = D / 8;         // bytes of a value row per lane
    constexpr int VP = VB >= 16 ? 16 : 8;
    constexpr int VC = VB / VP;       // pieces of a value row per lane
    constexpr int VW = VB / 4;        // words of a value row per lane
    constexpr int MT = D / 16;        // tiles of 16 d of O^T
    constexpr int KK = D / 16;        // k-steps of the dot product
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];
    __shared__ int join_count, join_done;  // shares left of the segment, and segments joined
    __shared__ int64_t scan[kWarps];
    if (threadIdx.x == 0) join_count = join_done = 0;  // ordered by the plan's barriers

    griddep_wait();
    griddep_launch_dependents();  // the join waits for this grid's end; its CTAs only become resident early

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int heads = a.c.kv_heads, batch = a.b.batch;

    // The plan: where each sequence's steps begin in the list, and the steps
    // of its segments. Sequences of more than max_rows rows are left to the
    // other kernel (no segments).
    int64_t *plan_first = reinterpret_cast<int64_t *>(smem + S::kRing + S::kJoin);  // [batch + 1]
    int *plan_steps = reinterpret_cast<int *>(plan_first + kMaxBatch + 1);                     // [batch]
    {
        int64_t total = 0;
        for (int s0 = 0; s0 < batch; s0 += kThreads) {
            const int s = s0 + threadIdx.x;
            int64_t mine = 0;
            if (s < batch) {
                const Span p = span_of<kRows, S::kPad>(a, s);
                if (p.cut && blockIdx.x == 0) record_device_error(a.err, kDevBadBatch);
                if (static_cast<int64_t>(p.n) * a.group <= max_rows) mine = static_cast<int64_t>(p.tiles) * heads * p.steps;
                plan_steps[s] = p.steps;
            }
            int64_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (lane == 31) scan[warp] = incl;
            __syncthreads();
            int64_t before = total, all = total;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) before += scan[w];
                all += scan[w];
            }
            if (s < batch) plan_first[s] = before + incl - mine;
            total = all;
            __syncthreads();
        }
        if (threadIdx.x == 0) plan_first[batch] = total;
        __syncthreads();
    }
    const int64_t total = plan_first[batch];
    // the sequence whose steps hold position p of the list
    auto sequence_at = [&](int64_t p) {
        int lo = 0, hi = batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (plan_first[mid] <= p) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    int64_t range = (total + gridDim.x - 1) / gridDim.x;
    if (range < S::kMinRange && !whole) range = S::kMinRange;
    int64_t from = range * blockIdx.x, to = min(from + range, total);
    if (whole && from < total) {  // segments that begin in the stretch, entirely
        auto up = [&](int64_t p) {  // the first segment boundary at or after p
            if (p >= total) return total;
            const int s = sequence_at(p);
            const int64_t in = p - plan_first[s], st = plan_steps[s];
            return plan_first[s] + (in + st - 1) / st * st;
        };
        from = up(from);
        to = up(to);
    }
    if (from >= to) {
        if (join_items != nullptr && threadIdx.x == 0) join_items[blockIdx.x].pieces = 0;
        return;
    }

    // Look-ups of 32 steps at a time, one step per lane: row of the cache
    // (-1: nothing to load), slots that hold a token, key scale, value scale
    // (0: no row sees the step).
    const int page_size = a.c.page_size, blk = a.c.scale_block;
    const int span = static_cast<int>(to - from);  // positions below are relative to `from`
    const int count = span > warp ? (span - warp + kWarps - 1) / kWarps : 0;  // this warp's steps
    struct Look {
        int row, held;
        float k, v;
    };
    auto look_up = [&](int i0) {
        Look r{-1, 0, 0.0f, 0.0f};
        const int i = i0 + lane;
        if (i < count) {
            const int64_t p = from + warp + static_cast<int64_t>(i) * kWarps;
            const int s = sequence_at(p);
            const int steps = plan_steps[s];
            const int64_t in = p - plan_first[s];
            const int th = in <= 0x7fffffff ? static_cast<int>(in) / steps : static_cast<int>(in / steps);  // 64-bit division is slow
            const int st = static_cast<int>(in - static_cast<int64_t>(th) * steps);
            const int tile = th / heads, head = th - tile * heads;
            const Span sp = span_of<kRows, S::kPad>(a, s);
            const int key = sp.lo + st * kStep;
            const int row_a = tile * kRows / a.group, row_z = (min(tile * kRows + kRows, sp.n * a.group) - 1) / a.group;
            const int hi = a.causal ? min(sp.pos0 + row_z, sp.len - 1) : sp.len - 1, lo = a.window > 0 ? sp.pos0 + row_a - a.window + 1 : 0;
            if (key <= hi && key + kStep > lo) {
                const int col = key / page_size, slot = key - col * page_size;
                const int64_t page = __ldg(a.b.block_table + s * a.b.table_stride + col);  // key < len <= the table's reach
                if (page >= 0 && page < a.c.num_pages) {
                    r.row = static_cast<int>((page * heads + head) * page_size + slot);
                    r.held = sp.len - key;
                    r.k = __ldg(a.c.k_scale + r.row / blk);
                    r.v = value_scale(__ldg(a.c.v_scale + r.row / blk));
                } else {
                    record_device_error(a.err, kDevBadPage);
                }
            }
        }
        return r;
    };

    const uint32_t ring = smem_u32(smem) + warp * (kStages * S::kStageBytes) + lane * 16;
    const uint32_t ring_v = smem_u32(smem) + warp * (kStages * S::kStageBytes) + kStep * D + lane * VP;
    const uint8_t *lane_k = a.c.k + g * D + c * 16, *lane_v = a.c.v + 2 * c * D + g * VB;
    uint32_t put = 0;  // byte offset of the ring stage the next issue fills
    Look cur, next = look_up(0);  // the batch being consumed, and the one being issued (the ring runs ahead by less than 32)
    auto issue = [&](int i) {
        const int row = __shfl_sync(0xffffffffu, next.row, i & 31), held = __shfl_sync(0xffffffffu, next.held, i & 31);
        if (row >= 0) {
            const int64_t off = static_cast<int64_t>(row) * D;
            const uint8_t *kp = lane_k + off, *vp = lane_v + off;
            if (held >= kStep) {
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int j = 0; j < KC; ++j) cp_async<16>(ring + put + (nt * KC + j) * 512, kp + nt * 8 * D + j * 64);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int j = 0; j < VC; ++j)
                        cp_async<VP>(ring_v + put + (t * VC + j) * (32 * VP), vp + ((t & 1) + (t >> 1) * 8) * D + j * VP);
            } else {  // the sequence's last step: zeros for the slots that hold nothing
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int j = 0; j < KC; ++j)
                        cp_async_zfill<16>(ring + put + (nt * KC + j) * 512, kp + nt * 8 * D + j * 64, g + 8 * nt < held ? 16u : 0u);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int j = 0; j < VC; ++j)
                        cp_async_zfill<VP>(ring_v + put + (t * VC + j) * (32 * VP), vp + ((t & 1) + (t >> 1) * 8) * D + j * VP,
                                           2 * c + (t & 1) + (t >> 1) * 8 < held ? VP : 0u);
            }
        }
        put = put == (kStages - 1) * S::kStageBytes ? 0 : put + S::kStageBytes;
        cp_async_commit();
    };

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    cur = next;  // not before: this waits for the scales
    uint32_t st = 0;  // the ring stage being consumed
    int i = 0;        // this warp's step

    int seq = sequence_at(from);
    int th = static_cast<int>((from - plan_first[seq]) / plan_steps[seq]);  // segment of the sequence: tile * heads + head
    int segment = 0;  // how many segments this CTA has left behind
    bool give_up = false;
    for (int at = 0; at < span;) {
        while (plan_first[seq + 1] <= from + at) {
            ++seq;
            th = 0;
        }
        const Span sp = span_of<kRows, S::kPad>(a, seq);
        const int tile = th / heads, head = th - tile * heads;
        const int seg = static_cast<int>(plan_first[seq] + static_cast<int64_t>(th) * sp.steps - from);  // the segment's first step
        const int end = min(seg + sp.steps, span);
        const int rows = min(kRows, sp.n * a.group - tile * kRows);

        // Q^T fragments: row g (+ 8), b0 and b1 the d of a key word's two pairs.
        // A lane's elements of a row are 16 consecutive ones of every 64. A
        // bf16 row is multiplied by a power of two first (exact), so its
        // largest element is in [1, 2) and fp16's range covers it.
        uint32_t qf[RG][KK][2];
        float fac[RG][2];  // of rows 2c, 2c + 1 (+ 8), as the scores lie
        int last[RG][2], first[RG][2];
        {
            const bool vec = aligned(a.q, 16) && a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) {
                const int r = g + 8 * rg, row = tile * kRows + r;
                uint32_t raw[KC][8];
#pragma unroll
                for (int j = 0; j < KC; ++j)
#pragma unroll
                    for (int w = 0; w < 8; ++w) raw[j][w] = 0;
                if (r < rows) {
                    const uint16_t *p = static_cast<const uint16_t *>(a.q) + (sp.t0 + static_cast<int64_t>(row / a.group)) * a.q_token_stride +
                                        (static_cast<int64_t>(head) * a.group + row % a.group) * a.q_head_stride + c * 16;
#pragma unroll
                    for (int j = 0; j < KC; ++j) {
                        if (vec) {
                            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p + j * 64)), v = __ldg(reinterpret_cast<const uint4 *>(p + j * 64) + 1);
                            raw[j][0] = u.x, raw[j][1] = u.y, raw[j][2] = u.z, raw[j][3] = u.w;
                            raw[j][4] = v.x, raw[j][5] = v.y, raw[j][6] = v.z, raw[j][7] = v.w;
                        } else {
#pragma unroll
                            for (int w = 0; w < 8; ++w) raw[j][w] = p[j * 64 + 2 * w] | (static_cast<uint32_t>(p[j * 64 + 2 * w + 1]) << 16);
                        }
                    }
                }
                float f = 1.0f;
                if (BF16) {
                    uint32_t mx = 0;
#pragma unroll
                    for (int j = 0; j < KC; ++j)
#pragma unroll
                        for (int w = 0; w < 8; ++w) mx = __vmaxu2(mx, raw[j][w] & 0x7fff7fffu);
                    mx = max(mx & 0xffffu, mx >> 16);
                    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    int e = static_cast<int>(mx >> 7);  // biased exponent of the row's largest element
                    e = mx == 0 ? 127 : min(max(e, 1), 253);
                    f = __uint_as_float(static_cast<uint32_t>(e) << 23);
                    const float inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
                    for (int j = 0; j < KC; ++j)
#pragma unroll
                        for (int w = 0; w < 8; ++w)
                            raw[j][w] = half2_bits(__uint_as_float(raw[j][w] << 16) * inv, __uint_as_float(raw[j][w] & 0xffff0000u) * inv);
                }
                f *= CAP ? a.inv_cap : a.scale_log2;
#pragma unroll
                for (int j = 0; j < KC; ++j)
#pragma unroll
                    for (int w = 0; w < 8; ++w) qf[rg][j * 4 + w / 2][w & 1] = raw[j][w];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    fac[rg][e] = __shfl_sync(0xffffffffu, f, (2 * c + e) * 4);
                    // rows past the tile's end (zero queries) see what its last row sees; they are not written
                    const int pos = sp.pos0 + (tile * kRows + min(8 * rg + 2 * c + e, rows - 1)) / a.group;
                    last[rg][e] = a.causal ? min(pos, sp.len - 1) : sp.len - 1;
                    first[rg][e] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
                }
            }
        }
        // keys in [all_lo, all_hi] are seen by every row of the tile
        const int row_a = tile * kRows / a.group, row_z = (tile * kRows + rows - 1) / a.group;
        const int all_hi = a.causal ? min(sp.pos0 + row_a, sp.len - 1) : sp.len - 1;
        const int all_lo = a.window > 0 ? max(0, sp.pos0 + row_z - a.window + 1) : 0;

        float o[RG][MT][4];  // O^T: d = g VB + 2 tile (+ 1 in 2, 3), rows 2c, 2c + 1
        float m[RG][2], l[RG][2];
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
            for (int t = 0; t < MT; ++t) o[rg][t][0] = o[rg][t][1] = o[rg][t][2] = o[rg][t][3] = 0.0f;
            m[rg][0] = m[rg][1] = -INFINITY;
            l[rg][0] = l[rg][1] = 0.0f;
        }
        bool first_step = true;  // some row has seen no key yet

        const int stop = end > warp ? (end - warp + kWarps - 1) / kWarps : 0;
        for (; i < stop; ++i) {
            if ((i & 31) == 0 && i > 0) cur = next;
            const int ahead = i + kStages - 1;
            if ((ahead & 31) == 0) next = look_up(ahead);
            issue(ahead);
            cp_async_wait<kStages - 1>();
            const uint32_t now = st;
            st = st == (kStages - 1) * S::kStageBytes ? 0 : st + S::kStageBytes;
            const float ks = __shfl_sync(0xffffffffu, cur.k, i & 31), vs = __shfl_sync(0xffffffffu, cur.v, i & 31);
            if (vs == 0.0f) continue;
            const int key = sp.lo + (warp + i * kWarps - seg) * kStep;
            // scores: keys g, g + 8 x rows 2c, 2c + 1 (+ 8)
            float x[RG][4];
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) x[rg][0] = x[rg][1] = x[rg][2] = x[rg][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                const uint4 k0 = lds128(ring + now + j * 512), k8 = lds128(ring + now + (KC + j) * 512);
                const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w8[4] = {k8.x, k8.y, k8.z, k8.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t af[4];
                    e4m3x4_to_half2(w0[q], af[0], af[2]);
                    e4m3x4_to_half2(w8[q], af[1], af[3]);
#pragma unroll
                    for (int rg = 0; rg < RG; ++rg) mma_f16(x[rg], af, qf[rg][j * 4 + q][0], qf[rg][j * 4 + q][1]);
                }
            }
            const float lvs = __log2f(vs), inv_vs = __fdividef(1.0f, vs);
            const bool edge = key < all_lo || key + kStep - 1 > all_hi;
            float e[RG][2][2], rows_sum[RG][2];  // weights [row][key g, g + 8]
            // Weights against the running reference maximum, which moves only
            // when a weight passes 2^8 (halves have room for that): no exchange
            // between lanes in most steps. The sum of a lane's weights bounds
            // each.
            bool again = edge || first_step;
            if (!again) {
                bool over = false;
#pragma unroll
                for (int rg = 0; rg < RG; ++rg)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float f = fac[rg][r] * ks, b = lvs - m[rg][r];
                        e[rg][r][0] = exp2_approx(CAP ? cap_score(x[rg][r], f, a.cap) + b : fmaf(x[rg][r], f, b));
                        e[rg][r][1] = exp2_approx(CAP ? cap_score(x[rg][2 + r], f, a.cap) + b : fmaf(x[rg][2 + r], f, b));
                        rows_sum[rg][r] = e[rg][r][0] + e[rg][r][1];
                        over |= rows_sum[rg][r] > 256.0f;
                    }
                again = __any_sync(0xffffffffu, over);
            }
            if (again) {
                bool over = false;
                float top[RG][2];
#pragma unroll
                for (int rg = 0; rg < RG; ++rg)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float f = fac[rg][r] * ks;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float y = CAP ? cap_score(x[rg][2 * k + r], f, a.cap) + lvs : fmaf(x[rg][2 * k + r], f, lvs);
                            const int at_key = key + g + 8 * k;
                            e[rg][r][k] = at_key <= last[rg][r] && at_key >= first[rg][r] ? y : -INFINITY;
                        }
                        float t = fmaxf(e[rg][r][0], e[rg][r][1]);
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                        top[rg][r] = t;
                        over |= t > m[rg][r] + (edge ? 8.0f : 0.0f);
                    }
                if (__any_sync(0xffffffffu, over)) {
                    bool seen = true;
#pragma unroll
                    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float to_m = fmaxf(m[rg][r], top[rg][r]);
                            const float f = to_m == m[rg][r] ? 1.0f : exp2_approx(m[rg][r] - to_m);  // 0 for the first keys
                            m[rg][r] = to_m;
                            l[rg][r] *= f;
#pragma unroll
                            for (int t = 0; t < MT; ++t) {
                                o[rg][t][r] *= f;
                                o[rg][t][2 + r] *= f;
                            }
                            seen &= to_m > -INFINITY;
                        }
                    first_step = !__all_sync(0xffffffffu, seen);
                }
#pragma unroll
                for (int rg = 0; rg < RG; ++rg)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float base = m[rg][r] == -INFINITY ? 0.0f : m[rg][r];  // nothing seen yet: 2^(-inf - 0) = 0
#pragma unroll
                        for (int k = 0; k < 2; ++k) e[rg][r][k] = exp2_approx(e[rg][r][k] - base);
                        rows_sum[rg][r] = e[rg][r][0] + e[rg][r][1];
                    }
            }
            uint32_t pf[RG][2];  // P^T fragments: row g, keys 2c, 2c + 1 (+ 8)
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
                for (int r = 0; r < 2; ++r) l[rg][r] = fmaf(rows_sum[rg][r], inv_vs, l[rg][r]);
                pf[rg][0] = transpose8x8(half2_bits(e[rg][0][0], e[rg][1][0]));
                pf[rg][1] = transpose8x8(half2_bits(e[rg][0][1], e[rg][1][1]));
            }
            // values: words of keys 2c, 2c + 1, 2c + 8, 2c + 9, paired per d
            uint32_t v[4][VW];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < VC; ++j) {
                    if constexpr (VP == 16) {
                        const uint4 u = lds128(ring_v + now + (t * VC + j) * 512);
                        v[t][j * 4] = u.x;
                        v[t][j * 4 + 1] = u.y;
                        v[t][j * 4 + 2] = u.z;
                        v[t][j * 4 + 3] = u.w;
                    } else {
                        const uint2 u = lds64(ring_v + now + t * 256);
                        v[t][0] = u.x;
                        v[t][1] = u.y;
                    }
                }
            // bytes 2h, 2h + 1 of word w: d of tile 2w + h
            auto value_tile = [&](const uint32_t(&from_v)[4][VW], int w, int h, uint32_t(&af)[4]) {
                e4m3x4_to_half2(__byte_perm(from_v[0][w], from_v[1][w], h ? 0x7362u : 0x5140u), af[0], af[1]);
                e4m3x4_to_half2(__byte_perm(from_v[2][w], from_v[3][w], h ? 0x7362u : 0x5140u), af[2], af[3]);
            };
            if (edge) {
                // A NaN among the values of a key that some row does not see
                // must not reach that row through 0 * NaN: count, per row and
                // d, the seen keys with a NaN there, and clear the codes.
                uint32_t any = 0;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int w = 0; w < VW; ++w) any |= nan_ones(v[t][w]);
                if (__any_sync(0xffffffffu, any != 0)) {
                    uint32_t ones[4][VW];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            ones[t][w] = nan_ones(v[t][w]);
                            v[t][w] = nan_cleared(v[t][w]);
                        }
#pragma unroll
                    for (int rg = 0; rg < RG; ++rg) {
                        const int pos = sp.pos0 + (tile * kRows + min(8 * rg + g, rows - 1)) / a.group;
                        const int hi = a.causal ? min(pos, sp.len - 1) : sp.len - 1, lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
                        float see[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int at_key = key + 2 * c + (k & 1) + (k >> 1) * 8;
                            see[k] = at_key <= hi && at_key >= lo ? 1.0f : 0.0f;
                        }
                        const uint32_t s0 = half2_bits(see[0], see[1]), s1 = half2_bits(see[2], see[3]);
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            uint32_t af[4];
                            float count_nan[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            value_tile(ones, t / 2, t % 2, af);
                            mma_f16(count_nan, af, s0, s1);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (count_nan[k] > 0.0f) o[rg][t][k] = NAN;
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t af[4];
                value_tile(v, t / 2, t % 2, af);
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) mma_f16(o[rg][t], af, pf[rg][0], pf[rg][1]);
            }
        }

        // Leave this warp's share, m, l and the valid rows of O, once the last
        // segment's have been joined (after a wait that was given up nothing
        // more is left or written).
        if constexpr (RG == 1) give_up = give_up || !wait_for(&join_done, segment, a.err);
        float4 *share = reinterpret_cast<float4 *>(smem + S::kRing) + warp * (S::kShare / 4);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[rg][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int r = 8 * rg + 2 * c + e;
                if (r < rows && !give_up) {
                    if (g == 0) {
                        join_m[warp][r] = m[rg][e];
                        join_l[warp][r] = sum;
                    }
#pragma unroll
                    for (int k = 0; k < MT / 2; ++k)
                        share[share_chunk<D>(r, g * (MT / 2) + k)] =
                            make_float4(o[rg][2 * k][e], o[rg][2 * k][2 + e], o[rg][2 * k + 1][e], o[rg][2 * k + 1][2 + e]);
                }
            }
        __threadfence_block();
        __syncwarp();
        // 8 rows: the last warp to come joins the shares, in warp order, while
        // the others go on. 16 rows would keep it too long: all warps join two
        // rows each.
        int before = 0;
        if constexpr (RG == 1) {
            if (lane == 0 && !give_up) before = atomicAdd(&join_count, 1);
            before = __shfl_sync(0xffffffffu, before, 0);
        } else {
            __syncthreads();
        }
        if (RG == 2 || before == kWarps - 1) {
            __threadfence_block();
            const bool cut = seg < 0 || seg + sp.steps > span;
            const float4 *all = reinterpret_cast<const float4 *>(smem + S::kRing);
            constexpr int LPR = D / 4 < 32 ? D / 4 : 32, RPW = 32 / LPR, CPL = D / 4 / LPR;  // lanes per row, rows at once, chunks per lane
            for (int r0 = RG == 1 ? 0 : warp * RPW; r0 < rows; r0 += RG == 1 ? RPW : kWarps * RPW) {
                const int r = r0 + lane / LPR;
                if (r < rows) {
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_m[w][r]);
                    float sum = 0.0f;
                    float4 acc[CPL];
#pragma unroll
                    for (int k = 0; k < CPL; ++k) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float wt = join_m[w][r] == -INFINITY ? 0.0f : exp2_approx(join_m[w][r] - top);
                        sum = fmaf(wt, join_l[w][r], sum);
#pragma unroll
                        for (int k = 0; k < CPL; ++k) {
                            const float4 v = all[w * (S::kShare / 4) + share_chunk<D>(r, k * LPR + lane % LPR)];
                            acc[k].x = fmaf(wt, v.x, acc[k].x);
                            acc[k].y = fmaf(wt, v.y, acc[k].y);
                            acc[k].z = fmaf(wt, v.z, acc[k].z);
                            acc[k].w = fmaf(wt, v.w, acc[k].w);
                        }
                    }
                    const int row = tile * kRows + r;
                    const int64_t token = sp.t0 + row / a.group;
                    const int qh = head * a.group + row % a.group;
                    const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (seg < 0 ? 0 : 1)) * part_rows + r;
                    const float inv = 1.0f / sum;
#pragma unroll
                    for (int k = 0; k < CPL; ++k) {
                        const int d0 = (k * LPR + lane % LPR) * 4;
                        if (cut) {
                            *reinterpret_cast<float4 *>(part_o + slot * D + d0) = acc[k];
                        } else {
                            const float y[4] = {acc[k].x, acc[k].y, acc[k].z, acc[k].w};
                            const int64_t off = token * a.out_token_stride + qh * a.out_head_stride + d0;
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const float z = sum != 0.0f ? y[t] * inv : 0.0f;  // NaN sums stay NaN
                                if (BF16) static_cast<__nv_bfloat16 *>(a.out)[off + t] = __float2bfloat16_rn(z);
                                else static_cast<__half *>(a.out)[off + t] = __float2half_rn(z);
                            }
                        }
                    }
                    if (lane % LPR == 0) {
                        if (cut) {
                            part_ml[slot * 2] = top;
                            part_ml[slot * 2 + 1] = sum;
                        } else if (a.lse != nullptr) {
                            a.lse[token * (static_cast<int64_t>(heads) * a.group) + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + log2f(sum));
                        }
                    }
                }
            }
            if constexpr (RG == 1) {
                __threadfence_block();
                __syncwarp();
                if (lane == 0) {
                    join_count = 0;
                    __threadfence_block();
                    *const_cast<volatile int *>(&join_done) = segment + 1;
                }
            } else {
                __syncthreads();
            }
        }
        // The CTA in which a cut segment begins names it to the join.
        if (join_items != nullptr && threadIdx.x == 0 && end == span) {
            JoinItem it{0, rows, tile * kRows, sp.t0, head, {0, 0, 0}};
            if (seg >= 0 && seg + sp.steps > span) it.pieces = static_cast<int>((from + seg + sp.steps - 1) / range) - static_cast<int>(blockIdx.x) + 1;
            join_items[blockIdx.x] = it;
        }
        at = end;
        ++th;
        ++segment;
    }
    cp_async_wait<0>();
}

// Merges the pieces of one row of a cut segment: grid (CTAs of the streaming
// kernel) x rows, 128 threads = 4 groups of pieces x 32 runs of columns.
template <int D, int RG>
__global__ void __launch_bounds__(128) k_kv_attention_join(AttnArgs a, int part_rows, const JoinItem *items, const float *part_ml,
                                                           const float *part_o) {
    griddep_launch_dependents();
    griddep_wait();
    const JoinItem it = items[blockIdx.x];
    const int r = blockIdx.y;
    if (it.pieces == 0 || r >= it.rows) return;
    constexpr int E = D / 32, kAhead = 8;
    __shared__ float red[4][D];
    __shared__ float red_m[4], red_l[4];
    const int part = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the first CTA's piece began with the segment (slot 1), the others' before their stretch (slot 0)
    auto at = [&](int k) { return (2 * (static_cast<int64_t>(blockIdx.x) + k) + (k == 0 ? 1 : 0)) * part_rows + r; };
    // warp `part` takes pieces part, part + 4, ..., several loads in flight, with a running maximum
    float top = -INFINITY, acc[E], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = 0.0f;
    for (int k0 = part; k0 < it.pieces; k0 += 4 * kAhead) {
        float2 ml[kAhead];
        float t[kAhead][E];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = k0 + 4 * u;
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (k < it.pieces) {
                ml[u] = *reinterpret_cast<const float2 *>(part_ml + at(k) * 2);
                load_vec<float, E>(part_o + at(k) * D + lane * E, t[u]);
            }
        }
        float next = top;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) next = fmaxf(next, ml[u].x);
        const float f = next == top ? 1.0f : exp2_approx(top - next);
        top = next;
        sum *= f;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] *= f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (k0 + 4 * u >= it.pieces) break;
            const float w = ml[u].x == -INFINITY ? 0.0f : exp2_approx(ml[u].x - top);
            sum = fmaf(w, ml[u].y, sum);
#pragma unroll
            for (int j = 0; j < E; ++j) acc[j] = fmaf(w, t[u][j], acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) red[part][lane * E + j] = acc[j];
    if (lane == 0) {
        red_m[part] = top;
        red_l[part] = sum;
    }
    __syncthreads();
    top = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    float wt[4];
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        wt[k] = red_m[k] == -INFINITY ? 0.0f : exp2_approx(red_m[k] - top);
        sum = fmaf(wt[k], red_l[k], sum);
    }
    const int row = it.row0 + r;
    const int64_t token = it.t0 + row / a.group;
    const int qh = it.head * a.group + row % a.group;
    const float inv = 1.0f / sum;
    for (int d = threadIdx.x; d < D; d += 128) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) v = fmaf(wt[k], red[k][d], v);
        const float y = sum != 0.0f ? v * inv : 0.0f;
        const int64_t off = token * a.out_token_stride + qh * a.out_head_stride + d;
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[off] = __float2bfloat16_rn(y);
        else static_cast<__half *>(a.out)[off] = __float2half_rn(y);
    }
    if (a.lse != nullptr && threadIdx.x == 0)
        a.lse[token * (static_cast<int64_t>(a.c.kv_heads) * a.group) + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + log2f(sum));
}

// What the host knows without the lengths.
struct Plan {
    int groups;     // of 8 rows per tile
    int grid;       // CTAs
    bool whole;     // no sequence reaches kWholeSteps: whole segments, no join
    int part_rows;  // rows of a piece in the workspace
    int64_t items, ml, o, bytes;  // workspace layout
};

Plan make_plan(const lcml_kv_attention_desc *d, int max_rows) {
    const lcml_kv_cache *c = d->cache;
    int64_t most = d->max_tokens < d->batch->total_tokens ? d->max_tokens : d->batch->total_tokens;
    most *= d->q_heads / c->kv_heads;
    if (most > max_rows) most = max_rows;
    if (most < 1) most = 1;
    Plan p{};
    p.groups = most <= 8 || c->head_dim == 256 ? 1 : 2;
    p.grid = sm_count() * stream_ctas(c->head_dim, p.groups);
    const int64_t reach = static_cast<int64_t>(d->batch->table_cols) * c->page_size;  // no sequence is longer
    p.whole = (reach + kStep - 1) / kStep <= kWholeSteps;
    if (p.whole) return p;
    p.part_rows = static_cast<int>(most < 8 * p.groups ? most : 8 * p.groups);
    const int64_t rows = 2 * static_cast<int64_t>(p.grid) * p.part_rows;
    p.items = 0;
    p.ml = (p.grid * static_cast<int64_t>(sizeof(JoinItem)) + 15) / 16 * 16;
    p.o = (p.ml + rows * 8 + 15) / 16 * 16;
    p.bytes = p.o + rows * c->head_dim * 4;
    return p;
}

template <int D, int RG>
int launch_stream(const lcml_kv_attention_desc *d, const AttnArgs &args, const Plan &p, int max_rows, cudaStream_t st) {
    using S = Shape<D, RG>;
    uint8_t *ws = static_cast<uint8_t *>(d->workspace);
    JoinItem *items = p.whole ? nullptr : reinterpret_cast<JoinItem *>(ws + p.items);
    float *ml = p.whole ? nullptr : reinterpret_cast<float *>(ws + p.ml);
    float *o = p.whole ? nullptr : reinterpret_cast<float *>(ws + p.o);
    auto kern = args.bf16 ? (args.cap != 0.0f ? k_kv_attention<D, RG, true, true> : k_kv_attention<D, RG, true, false>)
                          : (args.cap != 0.0f ? k_kv_attention<D, RG, false, true> : k_kv_attention<D, RG, false, false>);
    int rc = ensure_max_smem(reinterpret_cast<const void *>(kern), S::kSmem, "kv_attention");
    for (int64_t b0 = 0; rc == LCML_OK && b0 < d->batch->batch; b0 += kMaxBatch) {
        AttnArgs a = args;
        const int64_t n = d->batch->batch - b0;
        a.b.batch = static_cast<int32_t>(n < kMaxBatch ? n : kMaxBatch);
        a.b.cu_tokens += b0;
        a.b.lengths += b0;
        a.b.block_table += b0 * a.b.table_stride;
        rc = launch_dependent(kern, dim3(static_cast<unsigned>(p.grid)), S::kThreads, S::kSmem, st, "kv_attention", a, max_rows, p.whole, p.part_rows,
                              items, ml, o);
        if (rc == LCML_OK && !p.whole)
            rc = launch_dependent(k_kv_attention_join<D, RG>, dim3(static_cast<unsigned>(p.grid), static_cast<unsigned>(p.part_rows)), 128, 0, st,
                                  "kv_attention_join", a, p.part_rows, items, ml, o);
    }
    return rc;
}

int check_attention(const lcml_kv_attention_desc *d) {
    LCML_CHECK_ARG(d != nullptr, "lcml_kv_attention: null descriptor");
    int rc = check_cache(d->cache, "lcml_kv_attention");
    if (rc == LCML_OK) rc = check_batch(d->batch, "lcml_kv_attention");
    if (rc != LCML_OK) return rc;
    LCML_CHECK_ARG(d->dtype == LCML_DTYPE_FLOAT16 || d->dtype == LCML_DTYPE_BFLOAT16, "lcml_kv_attention: dtype %d unsupported", d->dtype);
    LCML_CHECK_ARG(d->q_heads > 0 && d->q_heads % d->cache->kv_heads == 0 && d->q_heads <= 65536,
                   "lcml_kv_attention: q_heads %d is not a multiple of kv_heads %d", d->q_heads, d->cache->kv_heads);
    LCML_CHECK_ARG(d->max_tokens >= 0, "lcml_kv_attention: negative max_tokens");
    LCML_CHECK_ARG(d->softmax_scale == d->softmax_scale && d->softcap >= 0.0f && d->window >= 0,
                   "lcml_kv_attention: softmax_scale is NaN, or softcap or window is negative");
    LCML_CHECK_ARG(d->window == 0 || d->causal, "lcml_kv_attention: a window needs causal");
    LCML_CHECK_ARG(d->variant >= 0 && d->variant <= 2, "lcml_kv_attention: variant %d", d->variant);
    return LCML_OK;
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" {

int64_t lcml_kv_attention_workspace_size(const lcml_kv_attention_desc *d) {
    if (check_attention(d) != LCML_OK) return -1;
    if (d->batch->batch == 0 || d->batch->total_tokens == 0) return 0;
    return make_plan(d, 0x7fffffff).bytes;
}

int lcml_kv_attention(const lcml_kv_attention_desc *d, lcml_stream_t stream) {
    const int rc = check_attention(d);
    if (rc != LCML_OK) return rc;
    if (d->batch->batch == 0 || d->batch->total_tokens == 0) return LCML_OK;
    LCML_CHECK_ARG(d->q && d->out, "lcml_kv_attention: null pointer");
    LCML_CHECK_ARG(aligned(d->q, 2) && aligned(d->out, 2) && aligned(d->lse, 4), "lcml_kv_attention: a pointer is not aligned to its element size");
    LCML_CHECK_ARG(d->q_token_stride >= 0 && d->q_head_stride >= 0 && d->out_token_stride >= 0 && d->out_head_stride >= 0,
                   "lcml_kv_attention: negative stride");
    // Rows of out are written by different CTAs: either stride covers the rows of the other.
    const int64_t tokens = d->batch->total_tokens, heads = d->q_heads, dim = d->cache->head_dim;
    const int64_t ts = d->out_token_stride, hs = d->out_head_stride;
    LCML_CHECK_ARG((tokens == 1 || ts >= dim) && (heads == 1 || hs >= dim) &&
                       (tokens == 1 || heads == 1 || ts >= (heads - 1) * hs + dim || hs >= (tokens - 1) * ts + dim),
                   "lcml_kv_attention: rows of out overlap (strides %lld and %lld)", (long long)ts, (long long)hs);
    const int64_t need = make_plan(d, 0x7fffffff).bytes;
    LCML_CHECK_ARG(need == 0 || (d->workspace && aligned(d->workspace, 16)), "lcml_kv_attention: needs a 16-byte aligned workspace of %lld bytes",
                   (long long)need);
    // No sequence is longer than its table reaches: a window of that many hides
    // nothing, and without it the kernels' position - window keeps to 32 bits.
    const int64_t reach = static_cast<int64_t>(d->batch->table_cols) * d->cache->page_size;
    AttnArgs a{*d->cache,         *d->batch,          d->q,
               d->out,            d->q_token_stride,  d->q_head_stride,
               d->out_token_stride, d->out_head_stride, d->lse,
               d->q_heads / d->cache->kv_heads, d->dtype == LCML_DTYPE_BFLOAT16, d->softmax_scale * kLog2e,
               d->softcap,        d->softcap > 0.0f ? d->softmax_scale / d->softcap : 0.0f, d->window < reach ? d->window : 0,
               d->causal ? 1 : 0, d->max_tokens,      device_error_word()};
    cudaStream_t st = to_cuda(stream);
    // Rows a sequence must have for the tensor-core kernel; the streaming
    // kernel takes the others. One launch where the bound or the variant says
    // that one kernel serves every sequence.
    const bool fits = kv_attention_tc_fits(d);
    LCML_CHECK_ARG(d->variant != 2 || fits, "lcml_kv_attention: variant 2 does not serve this call");
    const int64_t most = (d->max_tokens < d->batch->total_tokens ? d->max_tokens : d->batch->total_tokens) * a.group;
    int min_rows = 0x7fffffff;
    if (d->variant == 2) {
        min_rows = 1;
    } else if (fits && d->variant == 0) {
        const int rows = tc_rows(d->cache->head_dim);
        const int64_t all = d->batch->total_tokens * a.group;
        // units of the sequences with at least `rows` rows, at most
        const int64_t units = (all / kTcBlockRows + (d->batch->batch < all / rows ? d->batch->batch : all / rows)) * d->cache->kv_heads;
        if (most >= rows && all * d->cache->kv_heads >= rows * (units > sm_count() ? units : sm_count())) min_rows = rows;
    }
    if (min_rows != 0x7fffffff) {
        // If cu_tokens[batch] is total_tokens, the shortest sequence has at
        // least what the others, at max_tokens each, leave. A padded batch may
        // hold shorter ones all the same, so the kernel that runs alone takes
        // every sequence, however few its rows.
        const int64_t least = (d->batch->total_tokens - (d->batch->batch - 1) * static_cast<int64_t>(d->max_tokens)) * a.group;
        const bool alone = d->variant == 2 || least >= min_rows;
        const int rc2 = kv_attention_tc(d, a, alone ? 0 : min_rows, st);
        if (rc2 != LCML_OK || alone) return rc2;
    }
    const int max_rows = min_rows == 0x7fffffff ? min_rows : min_rows - 1;
    const Plan p = make_plan(d, max_rows);
    switch (d->cache->head_dim) {
        case 64: return p.groups == 1 ? launch_stream<64, 1>(d, a, p, max_rows, st) : launch_stream<64, 2>(d, a, p, max_rows, st);
        case 128: return p.groups == 1 ? launch_stream<128, 1>(d, a, p, max_rows, st) : launch_stream<128, 2>(d, a, p, max_rows, st);
        default: return launch_stream<256, 1>(d, a, p, max_rows, st);
    }
}

}// extern "C"
