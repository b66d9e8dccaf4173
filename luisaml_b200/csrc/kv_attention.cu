// Attention over the paged e4m3 cache: the streaming kernel (decode steps and
// short runs of queries) and the entry points.
//
// Rows of a sequence and cache head are its n queries x group heads, r = query
// * group + head, in tiles of 16 (the M of mma.m16n8k16). A CTA takes one row
// tile and a run of keys; its warps take every kWarps-th step of 16 keys, each
// with its own online softmax, and join at the end. Keys and values go from
// global memory through a per-lane cp.async ring straight into the fragment
// layout: the dot product's order of d is free, so a lane's key fragments are
// 16 consecutive bytes of one key row, and a value's output column is free
// too, so a lane reads consecutive bytes of four value rows and pairs them by
// byte permutes. Every lane reads back only what it copied itself: no
// barriers, no bank conflicts. Codes become halves by one exact conversion per
// pair; the block scales multiply the scores (keys) and join the exponent
// (values, value_scale()).
//
// Work split: the device-side plan cuts the batch into chunks of equal length
// such that about kTargetPerSm CTAs per SM exist whatever the lengths; rows
// with several chunks leave (m, l, O) partials that k_kv_attention_join merges
// in chunk order (deterministic).
//
// Bound: HBM, 2 head_dim bytes per key and cache head.
#include "lcml_attention.cuh"

namespace lcml {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;          // rows per tile
constexpr int kStep = 16;          // keys per warp step
constexpr int kMinChunk = 64;      // steps: below this a split costs more than it gains
constexpr int kTargetPerSm = 2;
constexpr int kTcRows = 128;       // rows of a sequence from which the tensor-core kernel takes it

template <int D>
struct Shape {
    static constexpr int kStages = D == 256 ? 2 : 4;
    static constexpr int kStageBytes = 2 * kStep * D;              // per warp
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kJoin = kWarps * kRows * D * 4;           // the warps' O, over the ring
    static constexpr int kQ = kRows * D * 2;                       // Q as half, fragment order
    static constexpr int kSmem = (kRing > kJoin ? kRing : kJoin) + kQ;
};

// Workspace: descriptors of the rows with several chunks, then partials.
struct JoinItem {
    int seq, tile, first_slot, chunks;
};

struct Plan {
    int64_t max_items;   // grid bound per head
    int64_t max_slots;   // partial slots per head
    int64_t max_joins;   // multi-chunk row tiles
    int target;          // chunk items aimed at per head
};

// Sequence b in steps of kStep keys: the visible span of a row tile differs
// between tiles only by less than the run of queries; the plan uses the
// sequence's whole span for all of its tiles.
struct Span {
    int n, len, lo, steps, tiles;
    int pos0;  // position of query 0 (negative: queries before the first token see nothing)
    bool cut;  // longer than the call's bounds
};

__device__ __forceinline__ Span span_of(const AttnArgs &a, int s) {
    Span r;
    const int t0 = __ldg(a.b.cu_tokens + s);
    const int t1 = static_cast<int>(min(static_cast<int64_t>(__ldg(a.b.cu_tokens + s + 1)), a.b.total_tokens));
    const int n = t0 >= 0 ? max(0, t1 - t0) : 0, len = max(0, __ldg(a.b.lengths + s));
    r.n = static_cast<int>(min(static_cast<int64_t>(n), a.max_tokens));
    r.len = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(a.b.table_cols) * a.c.page_size));
    r.cut = r.n < n || r.len < len;
    r.pos0 = r.len - n;
    const int64_t first = static_cast<int64_t>(r.pos0) - a.window + 1;  // the first query's oldest key
    r.lo = a.window > 0 && first > 0 ? static_cast<int>(first) & ~(kStep - 1) : 0;
    r.steps = (r.len - r.lo + kStep - 1) / kStep;
    r.tiles = static_cast<int>((static_cast<int64_t>(r.n) * a.group + kRows - 1) / kRows);
    return r;
}

__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What this CTA does: chunk `chunk` of row tile `tile` of sequence `seq`.
struct Item {
    int seq, tile, chunk, chunks, chunk_steps;
    int64_t slot;    // partial slot (chunks > 1)
    int64_t join;    // its row tile's index among those with several chunks
    int64_t joins;   // how many of those there are
    bool any;
};

// Every warp computes the plan for itself (a few coalesced loads and two
// passes over the batch): total work -> chunk length -> this item's place.
// Sequences of more than max_rows rows are left to the other kernel.
__device__ Item find_item(const AttnArgs &a, int64_t item, int target, int max_rows) {
    const int lane = threadIdx.x & 31;
    int64_t work = 0;
    for (int s = lane; s < a.b.batch; s += 32) {
        const Span p = span_of(a, s);
        if (p.cut) record_device_error(a.err, kDevBadBatch);
        if (static_cast<int64_t>(p.n) * a.group <= max_rows) work += static_cast<int64_t>(p.tiles) * p.steps;
    }
    work = warp_sum(work);
    Item r;
    r.any = false;
    const int64_t even = (work + target - 1) / target;
    const int c = static_cast<int>(even < kMinChunk ? kMinChunk : (even > 0x3fffffff ? 0x3fffffff : even));
    r.chunk_steps = c;
    int64_t items = 0, slots = 0, joins = 0;
    for (int s0 = 0; s0 < a.b.batch; s0 += 32) {
        int tiles = 0, chunks = 0;
        if (s0 + lane < a.b.batch) {
            const Span p = span_of(a, s0 + lane);
            if (static_cast<int64_t>(p.n) * a.group <= max_rows) {
                tiles = p.tiles;
                chunks = max(1, (p.steps + c - 1) / c);  // a sequence without keys still writes its zeros
            }
        }
        const int64_t mine = static_cast<int64_t>(tiles) * chunks;
        int64_t pi = mine, ps = chunks > 1 ? mine : 0, pj = chunks > 1 ? tiles : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, pi, o), y = __shfl_up_sync(0xffffffffu, ps, o),
                          z = __shfl_up_sync(0xffffffffu, pj, o);
            if (lane >= o) {
                pi += x;
                ps += y;
                pj += z;
            }
        }
        const bool here = !r.any && item < items + pi && mine > 0 && item >= items + pi - mine;
        const uint32_t who = __ballot_sync(0xffffffffu, here);
        if (who != 0) {
            const int src = __ffs(who) - 1;
            r.any = true;
            r.seq = s0 + src;
            r.chunks = __shfl_sync(0xffffffffu, chunks, src);
            const int64_t before = __shfl_sync(0xffffffffu, pi - mine, src);
            const int64_t sb = __shfl_sync(0xffffffffu, ps - (chunks > 1 ? mine : 0), src);
            const int64_t jb = __shfl_sync(0xffffffffu, pj - (chunks > 1 ? tiles : 0), src);
            const int64_t in = item - items - before;
            r.tile = static_cast<int>(in / r.chunks);
            r.chunk = static_cast<int>(in % r.chunks);
            r.slot = slots + sb + in;
            r.join = joins + jb + r.tile;
        }
        items += __shfl_sync(0xffffffffu, pi, 31);
        slots += __shfl_sync(0xffffffffu, ps, 31);
        joins += __shfl_sync(0xffffffffu, pj, 31);
    }
    r.joins = joins;
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

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
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

template <int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) k_kv_attention(AttnArgs a, int target, int max_rows, JoinItem *join_items, int *join_count,
                                                              float *part_ml, float *part_o) {
    using S = Shape<D>;
    constexpr int kStages = S::kStages;
    constexpr int KC = D / 64;        // 16-byte pieces of a key row per lane
    constexpr int VB = D / 8;         // bytes of a value row per lane
    constexpr int VP = VB >= 16 ? 16 : 8;
    constexpr int VC = VB / VP;       // pieces of a value row per lane
    constexpr int VW = VB / 4;        // words of a value row per lane
    constexpr int NT = D / 8;         // output tiles of 8 columns
    constexpr int KK = D / 16;        // k-steps of the dot product
    constexpr bool kQRegs = D <= 128;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float q_factor[kRows];
    __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];

    griddep_wait();
    griddep_launch_dependents();  // the join waits for this grid's end; its CTAs only become resident early

    const int head = blockIdx.x % a.c.kv_heads;
    const Item it = find_item(a, blockIdx.x / a.c.kv_heads, target, max_rows);
    if (blockIdx.x == 0 && threadIdx.x == 0 && join_count != nullptr) *join_count = static_cast<int>(it.joins);
    if (!it.any) return;
    const Span sp = span_of(a, it.seq);
    const int t0 = __ldg(a.b.cu_tokens + it.seq);
    if (it.chunks > 1 && it.chunk == 0 && head == 0 && threadIdx.x == 0)
        join_items[it.join] = JoinItem{it.seq, it.tile, static_cast<int>(it.slot), it.chunks};

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int rows = min(kRows, sp.n * a.group - it.tile * kRows);
    const int pos0 = sp.pos0;

    // Q tile -> halves in fragment order: word [(kk * 32 + lane) * 4 + reg]. A
    // bf16 row is multiplied by a power of two first (exact), so its largest
    // element is in [1, 2) and fp16's range covers it.
    uint32_t *qs = reinterpret_cast<uint32_t *>(smem + (S::kSmem - S::kQ));
    {
        constexpr int PER = D / 32;
        for (int r = warp; r < kRows; r += kWarps) {
            const int row = it.tile * kRows + r;
            float v[PER];
            uint32_t mx = 0;
            if (r < rows) {
                const int64_t off = (t0 + static_cast<int64_t>(row / a.group)) * a.q_token_stride +
                                    (static_cast<int64_t>(head) * a.group + row % a.group) * a.q_head_stride;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int d = lane * 2 + (j >> 1) * 64 + (j & 1);
                    v[j] = a.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[off + d])
                                  : __half2float(static_cast<const __half *>(a.q)[off + d]);
                    mx = max(mx, abs_bits_nan0(v[j]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) v[j] = 0.0f;
            }
            float f = 1.0f, inv = 1.0f;
            if (a.bf16) {
                mx = __reduce_max_sync(0xffffffffu, mx);
                int e = static_cast<int>(mx >> 23);             // biased exponent of the row's largest element
                e = mx == 0 ? 127 : min(max(e, 1), 253);
                f = __uint_as_float(static_cast<uint32_t>(e) << 23);
                inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
            }
            if (lane == 0) q_factor[r] = f;
#pragma unroll
            for (int j = 0; j < PER; j += 2) {
                const int d = lane * 2 + (j >> 1) * 64;  // even; d = i * 64 + cc * 16 + w * 4 + h * 2
                const int i = d >> 6, cc = (d >> 4) & 3, w = (d >> 2) & 3, h = (d >> 1) & 1;
                // a0: row g, first pair; a1: row g + 8, first pair; a2: row g, second pair; a3
                const int reg = h * 2 + (r >> 3), kk = i * 4 + w;
                qs[(kk * 32 + (r & 7) * 4 + cc) * 4 + reg] = half2_bits(v[j] * inv, v[j + 1] * inv);
            }
        }
    }
    __syncthreads();
    uint32_t qf[kQRegs ? KK : 1][4];
    if constexpr (kQRegs) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const uint4 t = lds128(smem_u32(qs + (kk * 32 + lane) * 4));
            qf[kk][0] = t.x;
            qf[kk][1] = t.y;
            qf[kk][2] = t.z;
            qf[kk][3] = t.w;
        }
    }

    // This lane's rows g and g + 8: score factor and the span of keys seen.
    float fac[2];
    int last[2], first[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        fac[i] = q_factor[r] * (CAP ? a.inv_cap : a.scale_log2);
        // rows past the tile's end (zero queries) see what its last row sees; they are not written
        const int pos = pos0 + (it.tile * kRows + min(r, rows - 1)) / a.group;
        last[i] = a.causal ? min(pos, sp.len - 1) : sp.len - 1;
        first[i] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    }
    // Over the tile: keys outside [tile_lo, tile_hi] are seen by no row, keys in [all_lo, all_hi] by every one.
    const int row_a = it.tile * kRows / a.group, row_z = (it.tile * kRows + rows - 1) / a.group;
    const int tile_hi = a.causal ? min(pos0 + row_z, sp.len - 1) : sp.len - 1;
    const int tile_lo = a.window > 0 ? max(0, pos0 + row_a - a.window + 1) : 0;
    const int all_hi = a.causal ? min(pos0 + row_a, sp.len - 1) : sp.len - 1;
    const int all_lo = a.window > 0 ? max(0, pos0 + row_z - a.window + 1) : 0;

    // Steps of this chunk that any row of the tile sees.
    int s_lo = it.chunk * it.chunk_steps;
    int s_hi = min(s_lo + it.chunk_steps, sp.steps);
    s_lo = max(s_lo, (tile_lo - sp.lo) / kStep);
    s_hi = min(s_hi, tile_hi < sp.lo ? 0 : (tile_hi - sp.lo) / kStep + 1);
    const int mine = s_hi - s_lo > warp ? (s_hi - s_lo - warp + kWarps - 1) / kWarps : 0;  // this warp's steps
    const int key0 = sp.lo + (s_lo + warp) * kStep;  // its i-th step starts at key0 + i * kWarps * kStep

    const int32_t *table = a.b.block_table + it.seq * a.b.table_stride;
    const int page_size = a.c.page_size, blk = a.c.scale_block;
    // Look-ups of 32 steps at a time, one step per lane: row of the cache
    // (-1: none), key scale, value scale.
    int look_row = -1;
    float look_k = 0.0f, look_v = 1.0f;
    auto look_up = [&](int i0) {
        look_row = -1;
        look_k = 0.0f;
        look_v = 1.0f;
        const int i = i0 + lane;
        if (i < mine) {
            const int key = key0 + i * (kWarps * kStep);
            const int col = key / page_size, slot = key - col * page_size;
            const int64_t page = col < a.b.table_cols ? __ldg(table + col) : -1;
            if (page >= 0 && page < a.c.num_pages) {
                const int row = static_cast<int>((page * a.c.kv_heads + head) * page_size + slot);
                look_row = row;
                look_k = __ldg(a.c.k_scale + row / blk);
                look_v = value_scale(__ldg(a.c.v_scale + row / blk));
            } else {
                record_device_error(a.err, kDevBadPage);
            }
        }
    };

    const uint32_t ring = smem_u32(smem) + warp * (kStages * S::kStageBytes) + lane * 16;
    const uint32_t ring_v = smem_u32(smem) + warp * (kStages * S::kStageBytes) + kStep * D + lane * VP;
    const uint8_t *lane_k = a.c.k + g * D + c * 16, *lane_v = a.c.v + 2 * c * D + g * VB;
    uint32_t put = 0;  // byte offset of the ring stage the next issue fills
    auto issue = [&](int i) {
        if (i < mine) {
            const int row = __shfl_sync(0xffffffffu, look_row, i & 31);
            const int held = row >= 0 ? sp.len - (key0 + i * (kWarps * kStep)) : 0;  // slots of the step that hold a token
            const int64_t off = static_cast<int64_t>(max(row, 0)) * D;
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

    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    bool first_step = true;  // some row has seen no key yet

    look_up(0);
    float use_k = look_k, use_v = look_v;  // the batch of look-ups being consumed (the ring runs ahead by less than 32)
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    uint32_t st = 0;  // the ring stage being consumed
    for (int i = 0; i < mine; ++i) {
        if ((i & 31) == 0 && i > 0) {
            use_k = look_k;
            use_v = look_v;
        }
        const int ahead = i + kStages - 1;
        if ((ahead & 31) == 0) look_up(ahead);
        issue(ahead);
        cp_async_wait<kStages - 1>();
        const float ks = __shfl_sync(0xffffffffu, use_k, i & 31), vs = __shfl_sync(0xffffffffu, use_v, i & 31);

        // scores: 16 rows x 16 keys; this lane: rows g, g + 8, keys 2c, 2c + 1 (+ 8)
        float x[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                const uint4 kv = lds128(ring + st + (nt * KC + j) * 512);
                const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t b0, b1;
                    e4m3x4_to_half2(w[q], b0, b1);
                    if constexpr (kQRegs) {
                        mma_f16(x[nt], qf[j * 4 + q], b0, b1);
                    } else {
                        const uint4 t = lds128(smem_u32(qs + ((j * 4 + q) * 32 + lane) * 4));
                        const uint32_t af[4] = {t.x, t.y, t.z, t.w};
                        mma_f16(x[nt], af, b0, b1);
                    }
                }
            }
        }
        const int key = key0 + i * (kWarps * kStep);
        const float lvs = __log2f(vs), inv_vs = __fdividef(1.0f, vs);
        const float f0 = fac[0] * ks, f1 = fac[1] * ks;
        const bool edge = key < all_lo || key + kStep - 1 > all_hi;
        float e[2][4], rows_sum[2];
        // Weights against the running reference maximum, which moves only when
        // a weight passes 2^8 (halves have room for that): no exchange between
        // lanes in most steps. The sum of a lane's weights bounds each.
        bool again = CAP || edge || first_step;
        if (!again) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = r ? f1 : f0, b = lvs - m[r];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[r][k] = exp2_approx(fmaf(x[k >> 1][2 * r + (k & 1)], f, b));
                rows_sum[r] = (e[r][0] + e[r][1]) + (e[r][2] + e[r][3]);
            }
            again = __any_sync(0xffffffffu, rows_sum[0] > 256.0f || rows_sum[1] > 256.0f);
        }
        if (again) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = r ? f1 : f0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float y = x[k >> 1][2 * r + (k & 1)];
                    y = CAP ? cap_score(y, f, a.cap) + lvs : fmaf(y, f, lvs);
                    const int at = key + (k >> 1) * 8 + 2 * c + (k & 1);
                    e[r][k] = at <= last[r] && at >= first[r] ? y : -INFINITY;
                    top[r] = fmaxf(top[r], e[r][k]);
                }
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] + (CAP || edge ? 8.0f : 0.0f) || top[1] > m[1] + (CAP || edge ? 8.0f : 0.0f))) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float to = fmaxf(m[r], top[r]);
                    const float f = to == m[r] ? 1.0f : exp2_approx(m[r] - to);  // 0 for the first keys
                    m[r] = to;
                    l[r] *= f;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        o[t][2 * r] *= f;
                        o[t][2 * r + 1] *= f;
                    }
                }
                first_step = !__all_sync(0xffffffffu, m[0] > -INFINITY && m[1] > -INFINITY);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float base = m[r] == -INFINITY ? 0.0f : m[r];  // nothing seen yet: 2^(-inf - 0) = 0
#pragma unroll
                for (int k = 0; k < 4; ++k) e[r][k] = exp2_approx(e[r][k] - base);
                rows_sum[r] = (e[r][0] + e[r][1]) + (e[r][2] + e[r][3]);
            }
        }
        uint32_t p[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] = fmaf(rows_sum[r], inv_vs, l[r]);
            p[r] = half2_bits(e[r][0], e[r][1]);
            p[2 + r] = half2_bits(e[r][2], e[r][3]);
        }
        // values: words of the lane's four keys, paired per output column
        uint32_t v[4][VW];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < VC; ++j) {
                if constexpr (VP == 16) {
                    const uint4 u = lds128(ring_v + st + (t * VC + j) * 512);
                    v[t][j * 4] = u.x;
                    v[t][j * 4 + 1] = u.y;
                    v[t][j * 4 + 2] = u.z;
                    v[t][j * 4 + 3] = u.w;
                } else {
                    const uint2 u = lds64(ring_v + st + t * 256);
                    v[t][0] = u.x;
                    v[t][1] = u.y;
                }
            }
        if (edge) {
            // A NaN among the values of a key that some row does not see must
            // not reach that row through 0 * NaN: count, per row and column,
            // the seen keys with a NaN there, and clear the codes.
            uint32_t any = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int w = 0; w < VW; ++w) any |= nan_ones(v[t][w]);
            if (__any_sync(0xffffffffu, any != 0)) {
                uint32_t see[4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float f[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = key + (k >> 1) * 8 + 2 * c + (k & 1);
                        f[k] = j <= last[r] && j >= first[r] ? 1.0f : 0.0f;
                    }
                    see[r] = half2_bits(f[0], f[1]);
                    see[2 + r] = half2_bits(f[2], f[3]);
                }
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const uint32_t n0 = nan_ones(v[0][w]), n1 = nan_ones(v[1][w]), n2 = nan_ones(v[2][w]), n3 = nan_ones(v[3][w]);
                    const uint32_t a0 = __byte_perm(n0, n1, 0x5140), a1 = __byte_perm(n0, n1, 0x7362);
                    const uint32_t b0 = __byte_perm(n2, n3, 0x5140), b1 = __byte_perm(n2, n3, 0x7362);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float cnt[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        const uint32_t wa = k < 2 ? a0 : a1, wb = k < 2 ? b0 : b1;
                        mma_f16(cnt, see, e4m3x2_to_half2((wa >> ((k & 1) * 16)) & 0xffffu), e4m3x2_to_half2((wb >> ((k & 1) * 16)) & 0xffffu));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (cnt[e] > 0.0f) o[w * 4 + k][e] = NAN;
                    }
#pragma unroll
                    for (int t = 0; t < 4; ++t) v[t][w] = nan_cleared(v[t][w]);
                }
            }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
            const uint32_t b0 = __byte_perm(v[2][w], v[3][w], 0x5140), b1 = __byte_perm(v[2][w], v[3][w], 0x7362);
            uint32_t ha[4], hb[4];
            e4m3x4_to_half2(a0, ha[0], ha[1]);
            e4m3x4_to_half2(a1, ha[2], ha[3]);
            e4m3x4_to_half2(b0, hb[0], hb[1]);
            e4m3x4_to_half2(b1, hb[2], hb[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_f16(o[w * 4 + k], p, ha[k], hb[k]);
        }
        st = st == (kStages - 1) * S::kStageBytes ? 0 : st + S::kStageBytes;
    }
    cp_async_wait<0>();

    // Join the warps: O in fragment order [warp][tile * 4 + reg][lane] over the ring.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (c == 0) {
            join_m[warp][g + 8 * r] = m[r];
            join_l[warp][g + 8 * r] = l[r];
        }
    }
    __syncthreads();  // every warp has left the ring
    float *os = reinterpret_cast<float *>(smem) + warp * (kRows * D);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) os[(t * 4 + e) * 32 + lane] = o[t][e];
    __syncthreads();

    // Thread = (half of the tiles, reg e, lane): NT / 2 consecutive output columns of one row.
    const int half = threadIdx.x >> 7, e = (threadIdx.x >> 5) & 3;
    const int r = g + 8 * (e >> 1);
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_m[w][r]);
    float wt[kWarps], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        wt[w] = join_m[w][r] == -INFINITY ? 0.0f : exp2_approx(join_m[w][r] - top);
        sum = fmaf(wt[w], join_l[w][r], sum);
    }
    float acc[NT / 2];
    const float *src = reinterpret_cast<const float *>(smem);
#pragma unroll
    for (int t = 0; t < NT / 2; ++t) {
        acc[t] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) acc[t] = fmaf(wt[w], src[w * (kRows * D) + ((half * (NT / 2) + t) * 4 + e) * 32 + lane], acc[t]);
    }
    if (r >= rows) return;
    const int d0 = (2 * c + (e & 1)) * VB + half * (NT / 2);
    if (it.chunks > 1) {
        const int64_t slot = it.slot * a.c.kv_heads + head;
        float *dst = part_o + (slot * kRows + r) * D + d0;
#pragma unroll
        for (int t = 0; t < NT / 2; t += 4) *reinterpret_cast<float4 *>(dst + t) = make_float4(acc[t], acc[t + 1], acc[t + 2], acc[t + 3]);
        if (half == 0 && (e & 1) == 0 && c == 0) {
            part_ml[(slot * kRows + r) * 2] = top;
            part_ml[(slot * kRows + r) * 2 + 1] = sum;
        }
        return;
    }
    const int row = it.tile * kRows + r;
    const int64_t token = t0 + row / a.group;
    const int qh = head * a.group + row % a.group;
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // NaN sums stay NaN
    const int64_t off = token * a.out_token_stride + qh * a.out_head_stride + d0;
#pragma unroll
    for (int t = 0; t < NT / 2; ++t) {
        const float y = sum != 0.0f ? acc[t] * inv : 0.0f;
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[off + t] = __float2bfloat16_rn(y);
        else static_cast<__half *>(a.out)[off + t] = __float2half_rn(y);
    }
    if (a.lse != nullptr && half == 0 && (e & 1) == 0 && c == 0)
        a.lse[token * (static_cast<int64_t>(a.c.kv_heads) * a.group) + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + log2f(sum));
}

// Merges the chunks of one row of a row tile: grid (row tiles with several
// chunks, at most) x heads x 16 rows, 128 threads = 4 groups of chunks x 32
// columns' vectors.
template <int D>
__global__ void __launch_bounds__(128) k_kv_attention_join(AttnArgs a, int max_slots, const JoinItem *items, const int *count,
                                                           const float *part_ml, const float *part_o) {
    griddep_launch_dependents();
    griddep_wait();
    if (static_cast<int>(blockIdx.x) >= *count) return;
    const JoinItem it = items[blockIdx.x];
    // cannot be otherwise for increasing cu_tokens
    if (it.seq < 0 || it.seq >= a.b.batch || it.tile < 0 || it.first_slot < 0 || it.chunks < 0 || it.first_slot > max_slots - it.chunks) return;
    const int head = blockIdx.y, r = blockIdx.z;
    const Span sp = span_of(a, it.seq);
    const int row = it.tile * kRows + r;
    if (row >= sp.n * a.group) return;
    constexpr int E = D / 32;
    __shared__ float red[4][D];
    __shared__ float red_l[4];
    const int part = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto at = [&](int ch) { return ((static_cast<int64_t>(it.first_slot) + ch) * a.c.kv_heads + head) * kRows + r; };
    float top = -INFINITY;
    for (int ch = lane; ch < it.chunks; ch += 32) top = fmaxf(top, part_ml[at(ch) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float acc[E], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = 0.0f;
    for (int ch = part; ch < it.chunks; ch += 4) {
        const float mc = part_ml[at(ch) * 2], lc = part_ml[at(ch) * 2 + 1];
        const float w = mc == -INFINITY ? 0.0f : exp2_approx(mc - top);
        sum = fmaf(w, lc, sum);
        const float *src = part_o + at(ch) * D + lane * E;
        float t[E];
        load_vec<float, E>(src, t);
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = fmaf(w, t[j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) red[part][lane * E + j] = acc[j];
    if (lane == 0) red_l[part] = sum;
    __syncthreads();
    sum = (red_l[0] + red_l[1]) + (red_l[2] + red_l[3]);
    const int64_t token = __ldg(a.b.cu_tokens + it.seq) + row / a.group;
    const int qh = head * a.group + row % a.group;
    const float inv = 1.0f / sum;
    for (int d = threadIdx.x; d < D; d += 128) {
        const float v = (red[0][d] + red[1][d]) + (red[2][d] + red[3][d]);
        const float y = sum != 0.0f ? v * inv : 0.0f;
        const int64_t off = token * a.out_token_stride + qh * a.out_head_stride + d;
        if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[off] = __float2bfloat16_rn(y);
        else static_cast<__half *>(a.out)[off] = __float2half_rn(y);
    }
    if (a.lse != nullptr && threadIdx.x == 0)
        a.lse[token * (static_cast<int64_t>(a.c.kv_heads) * a.group) + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + log2f(sum));
}

// Bounds the host can give without the lengths. Items per head: every row
// tile has at least one, and cutting the total work W into chunks of at least
// W / target steps adds at most target. Chunks of split row tiles: a tile
// with several chunks of c steps has at most 2 steps / c of them.
Plan make_plan(const lcml_kv_attention_desc *d, int max_rows) {
    const lcml_kv_cache *c = d->cache;
    const lcml_kv_batch *b = d->batch;
    const int group = d->q_heads / c->kv_heads;
    Plan p;
    p.target = (kTargetPerSm * sm_count() + c->kv_heads - 1) / c->kv_heads;
    int64_t most = d->max_tokens < b->total_tokens ? d->max_tokens : b->total_tokens;
    if (most * group > max_rows) most = max_rows / group;
    const int64_t per_seq = (most * group + kRows - 1) / kRows;
    int64_t tiles = b->total_tokens * group / kRows + b->batch;
    if (tiles > per_seq * b->batch) tiles = per_seq * b->batch;
    p.max_items = tiles + p.target;
    const int64_t reach = static_cast<int64_t>(b->table_cols) * c->page_size;  // no sequence is longer
    const bool never = (reach + kStep - 1) / kStep + 1 <= kMinChunk;
    p.max_slots = never ? 0 : 2 * static_cast<int64_t>(p.target) + 2;
    p.max_joins = never ? 0 : p.target + 1;
    return p;
}

struct Workspace {
    int64_t count, items, ml, o, bytes;
};

Workspace lay_out(const Plan &p, const lcml_kv_attention_desc *d) {
    Workspace w{};
    if (p.max_slots == 0) return w;
    const int64_t rows = p.max_slots * d->cache->kv_heads * kRows;
    w.count = 0;
    w.items = 16;
    w.ml = (w.items + p.max_joins * static_cast<int64_t>(sizeof(JoinItem)) + 15) / 16 * 16;
    w.o = w.ml + rows * 8;
    w.bytes = w.o + rows * d->cache->head_dim * 4;
    return w;
}

template <int D>
int launch_stream(const lcml_kv_attention_desc *d, const AttnArgs &a, int max_rows, cudaStream_t st) {
    const Plan p = make_plan(d, max_rows);
    const Workspace w = lay_out(p, d);
    uint8_t *ws = static_cast<uint8_t *>(d->workspace);
    JoinItem *items = p.max_slots ? reinterpret_cast<JoinItem *>(ws + w.items) : nullptr;
    int *count = p.max_slots ? reinterpret_cast<int *>(ws + w.count) : nullptr;
    float *ml = p.max_slots ? reinterpret_cast<float *>(ws + w.ml) : nullptr;
    float *o = p.max_slots ? reinterpret_cast<float *>(ws + w.o) : nullptr;
    LCML_CHECK_ARG(p.max_items * d->cache->kv_heads <= 0x7fffffff, "lcml_kv_attention: too much work for one call");
    auto kern = a.cap != 0.0f ? k_kv_attention<D, true> : k_kv_attention<D, false>;
    int rc = ensure_max_smem(reinterpret_cast<const void *>(kern), Shape<D>::kSmem, "kv_attention");
    if (rc != LCML_OK) return rc;
    rc = launch_dependent(kern, dim3(static_cast<unsigned>(p.max_items * d->cache->kv_heads)), kThreads, Shape<D>::kSmem, st,
                          "kv_attention", a, p.target, max_rows, items, count, ml, o);
    if (rc != LCML_OK || p.max_slots == 0) return rc;
    return launch_dependent(k_kv_attention_join<D>, dim3(static_cast<unsigned>(p.max_joins), d->cache->kv_heads, kRows), 128, 0, st,
                            "kv_attention_join", a, static_cast<int>(p.max_slots), items, count, ml, o);
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
    return lay_out(make_plan(d, 0x7fffffff), d).bytes;
}

int lcml_kv_attention(const lcml_kv_attention_desc *d, lcml_stream_t stream) {
    const int rc = check_attention(d);
    if (rc != LCML_OK) return rc;
    if (d->batch->batch == 0 || d->batch->total_tokens == 0) return LCML_OK;
    LCML_CHECK_ARG(d->q && d->out, "lcml_kv_attention: null pointer");
    LCML_CHECK_ARG(aligned(d->q, 2) && aligned(d->out, 2) && aligned(d->lse, 4), "lcml_kv_attention: a pointer is not aligned to its element size");
    LCML_CHECK_ARG(d->q_token_stride >= 0 && d->q_head_stride >= 0 && d->out_token_stride >= 0 && d->out_head_stride >= 0,
                   "lcml_kv_attention: negative stride");
    const int64_t need = lay_out(make_plan(d, 0x7fffffff), d).bytes;
    LCML_CHECK_ARG(need == 0 || (d->workspace && aligned(d->workspace, 16)), "lcml_kv_attention: needs a 16-byte aligned workspace of %lld bytes",
                   (long long)need);
    AttnArgs a{*d->cache,         *d->batch,          d->q,
               d->out,            d->q_token_stride,  d->q_head_stride,
               d->out_token_stride, d->out_head_stride, d->lse,
               d->q_heads / d->cache->kv_heads, d->dtype == LCML_DTYPE_BFLOAT16, d->softmax_scale * kLog2e,
               d->softcap,        d->softcap > 0.0f ? d->softmax_scale / d->softcap : 0.0f, d->window,
               d->causal ? 1 : 0, d->max_tokens,      device_error_word()};
    cudaStream_t st = to_cuda(stream);
    // Rows a sequence must have for the tensor-core kernel; the streaming
    // kernel takes the others. One launch where the bound or the variant says
    // that one kernel serves every sequence.
    const bool fits = kv_attention_tc_fits(d);
    LCML_CHECK_ARG(d->variant != 2 || fits, "lcml_kv_attention: variant 2 does not serve this call");
    const int64_t most = (d->max_tokens < d->batch->total_tokens ? d->max_tokens : d->batch->total_tokens) * a.group;
    int min_rows = fits && d->variant != 1 ? (d->variant == 2 ? 0 : kTcRows) : 0x7fffffff;
    if (most < min_rows) min_rows = 0x7fffffff;
    if (min_rows != 0x7fffffff) {
        const int rc2 = kv_attention_tc(d, a, min_rows, st);
        if (rc2 != LCML_OK || min_rows == 0 || d->batch->batch == 1) return rc2;
    }
    const int max_rows = min_rows == 0x7fffffff ? min_rows : min_rows - 1;
    switch (d->cache->head_dim) {
        case 64: return launch_stream<64>(d, a, max_rows, st);
        case 128: return launch_stream<128>(d, a, max_rows, st);
        default: return launch_stream<256>(d, a, max_rows, st);
    }
}

}// extern "C"
