// The plan of a ragged batch (lcml_kv_plan): pages given back and taken, block
// tables, positions and slots from request lengths.
//
// One launch of one cluster. Every CTA scans the whole batch for itself (the
// lengths of a few hundred rows are a handful of loads a thread), so the CTAs
// exchange only the counts of the pages that ended rows give back; then each
// takes a share of the table's new entries and of the tokens, and finds a
// token's row by a search in the sums that it holds in shared memory. A page that
// is taken is free_pages[count - 1 - i] for the i-th new entry of the batch, so
// entry and slots are computed apart, without a second pass over the table.
//
// Bound: latency. A step of 64 rows moves 2 KB: 2.8 us. 256 rows of which 26 end, 45,000 tokens: 11.7 us.
#include <type_traits>

#include "lcml_decoder.cuh"

#include "../../include/lcml_decode_step.h"

namespace lcml {
namespace {

constexpr int kDevNoPages = 8;  // joins the codes of DeviceError: the free list ran out
constexpr int kMaxRows = 16384;
constexpr int kThreads = 1024;  // at most
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kEntries = 8;  // of an ended row, that a lane loads at once
constexpr unsigned kAll = 0xffffffffu;

// Exclusive sums of two values a thread over the block; the totals are added to `tokens` and `entries`.
struct Scan {
    int64_t tokens[kWarps];
    int32_t entries[kWarps];
};
__device__ __forceinline__ void block_scan(Scan &sh, int64_t &a, int32_t &b, int64_t &tokens, int32_t &entries) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int64_t x = a;
    int32_t y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t p = __shfl_up_sync(kAll, x, o);
        const int32_t q = __shfl_up_sync(kAll, y, o);
        if (lane >= o) {
            x += p;
            y += q;
        }
    }
    if (lane == 31) {
        sh.tokens[warp] = x;
        sh.entries[warp] = y;
    }
    __syncthreads();
    // every warp sums the warps' sums
    int64_t before = lane < warps ? sh.tokens[lane] : 0, all = before;
    int32_t before_e = lane < warps ? sh.entries[lane] : 0;
    const int32_t all_e = __reduce_add_sync(kAll, before_e);
    before = lane < warp ? before : 0;
    before_e = __reduce_add_sync(kAll, lane < warp ? before_e : 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(kAll, before, o);
        all += __shfl_xor_sync(kAll, all, o);
    }
    before += tokens;
    before_e += entries;
    __syncthreads();
    a = before + x - a;
    b = before_e + y - b;
    tokens += all;
    entries += all_e;
}

// The last i in [0, n) with first[i] <= x; first[0] <= x, not decreasing.
__device__ __forceinline__ int last_at_or_below(const int32_t *first, int n, int x) {
    int lo = 0;
    for (int step = 1 << (31 - __clz(n | 1)); step > 0; step >>= 1)
        if (lo + step < n && first[lo + step] <= x) lo += step;
    return lo;
}

// n / page_size for n below 2^31: (n factor) >> shift, where 2^shift is 2^31 times the least power of two
// that is page_size or more and factor = floor(2^shift / page_size) + 1, too large by page_size / 2^shift at most.
struct PageDivision {
    uint32_t factor;
    int shift;
    explicit PageDivision(uint32_t page_size) : shift(31) {
        while ((1u << (shift - 31)) < page_size) ++shift;
        factor = static_cast<uint32_t>((uint64_t{1} << shift) / page_size + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return static_cast<uint32_t>(static_cast<uint64_t>(n) * factor >> shift); }
};

__global__ void __launch_bounds__(kThreads) k_kv_plan(lcml_kv_plan_desc a, PageDivision page_in, int *err) {
    extern __shared__ int32_t smem[];
    __shared__ Scan scan;
    const int batch = a.batch;
    int32_t *cu = smem;                  // [batch + 1]
    int32_t *shift = smem + batch + 1;   // [batch]: a token's position less its packed index
    int32_t *pages = shift + batch;      // [batch + 1]: new entries of the rows before; at first, pages given back
    const int lane = threadIdx.x & 31;
    const int ctas = gridDim.x, rank = blockIdx.x;
    const int stride = ctas * blockDim.x, me = rank * blockDim.x + threadIdx.x;
    const uint32_t ps = a.page_size;
    const int64_t reach = static_cast<int64_t>(a.table_cols) * ps;
    const int total = static_cast<int>(a.total_tokens);
    bool bad = false;

    if (a.ended != nullptr) {
        for (int b = threadIdx.x; b < batch; b += blockDim.x) pages[b] = 0;
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    }
    griddep_launch_dependents();
    griddep_wait();
    const int listed = *a.free_count;
    const int64_t capacity = a.free_capacity < 0x7fffffff ? a.free_capacity : 0x7fffffff;
    int64_t count = listed < 0 ? 0 : (listed < capacity ? listed : capacity);
    bad |= count != listed;

    auto columns = [&](int tokens) -> int {  // columns of the table that hold this many (>= 0)
        return tokens > 0 ? min(static_cast<int>(page_in(tokens - 1)) + 1, a.table_cols) : 0;
    };
    if (a.ended != nullptr) {
        // The rows are dealt to the cluster's warps, which take their ended ones in turn; a count goes to every CTA.
        auto row_entry = [&](int b, int c, int n) -> int { return c < n ? a.block_table[b * a.table_stride + c] : -1; };
        const int warps = stride >> 5, w = me >> 5;
        auto each_ended = [&](auto f) {
            for (int b0 = w; b0 < batch; b0 += 32 * warps) {
                const int b = b0 + lane * warps;
                const bool in = b < batch;
                const int cols = in ? columns(max(0, a.held[b])) : 0;
                for (uint32_t m = __ballot_sync(kAll, in && a.ended[in ? b : 0] != 0); m != 0; m &= m - 1) {
                    const int l = __ffs(m) - 1;
                    f(b0 + l * warps, __shfl_sync(kAll, cols, l));
                }
            }
        };
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every CTA has started
        each_ended([&](int b, int cols) {
            int n = 0;
            for (int c0 = 0; c0 < cols; c0 += 32 * kEntries) {
#pragma unroll
                for (int j = 0; j < kEntries; ++j) n += row_entry(b, c0 + 32 * j + lane, cols) >= 0;
            }
            n = __reduce_add_sync(kAll, n);
            if (lane < ctas) {
                const uint32_t to = mapa_shared(smem_u32(pages + b), lane);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(n) : "memory");
            }
        });
        cluster_sync_all();
        int64_t unused = 0;
        int32_t back = 0;
        for (int b0 = 0; b0 < batch; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            int64_t none = 0;
            int32_t mine = b < batch ? pages[b] : 0;
            block_scan(scan, none, mine, unused, back);
            if (b < batch) pages[b] = mine;
        }
        __syncthreads();
        each_ended([&](int b, int cols) {
            int64_t at = count + pages[b];
            for (int c0 = 0; c0 < cols; c0 += 32 * kEntries) {
                int p[kEntries];
#pragma unroll
                for (int j = 0; j < kEntries; ++j) p[j] = row_entry(b, c0 + 32 * j + lane, cols);
#pragma unroll
                for (int j = 0; j < kEntries; ++j) {
                    const uint32_t have = __ballot_sync(kAll, p[j] >= 0);
                    const int64_t to = at + __popc(have & ((1u << lane) - 1));
                    if (p[j] >= 0) {
                        if (to < capacity) a.free_pages[to] = p[j];
                        a.block_table[b * a.table_stride + c0 + 32 * j + lane] = -1;
                    }
                    at += __popc(have);
                }
            }
        });
        bad |= count + back > capacity;
        count = count + back < capacity ? count + back : capacity;
        __syncthreads();  // `pages` may be written again
    }

    // Sums of the tokens and of the new entries; these again where tokens are left out.
    int64_t tokens = 0;
    int32_t taken = 0;
    for (int turn = 0; turn < 2; ++turn) {
        const int64_t limit = turn == 0 ? INT64_MAX : total;
        tokens = 0;
        taken = 0;
        for (int b0 = 0; b0 < batch; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            int n = 0, start = 0;
            if (b < batch) {
                n = a.new_tokens[b];
                start = a.held[b];
                bad |= n < 0 || start < 0;
                n = max(n, 0);
                start = a.ended != nullptr && a.ended[b] != 0 ? 0 : max(start, 0);
            }
            int64_t first = n;
            if (turn == 1) n = static_cast<int>(min(static_cast<int64_t>(cu[b < batch ? b : 0]) + n, limit) - cu[b < batch ? b : 0]);  // cu: of turn 0
            const int64_t len = min(static_cast<int64_t>(start) + n, static_cast<int64_t>(0x7fffffff));
            bad |= b < batch && len > reach;
            int32_t entries = b < batch ? columns(static_cast<int>(len)) - columns(start) : 0;
            block_scan(scan, first, entries, tokens, taken);
            if (b < batch) {
                cu[b] = static_cast<int32_t>(min(first, static_cast<int64_t>(total)));
                shift[b] = start - cu[b];
                pages[b] = entries;
            }
        }
        if (tokens <= total) break;
        bad = true;
        __syncthreads();
    }
    if (threadIdx.x == 0) cu[batch] = static_cast<int32_t>(min(tokens, static_cast<int64_t>(total)));
    if (rank == 0 && bad) record_device_error(err, kDevBadBatch);
    // The free list is complete, and every CTA has read held and free_count: kv_len and free_count_out may be the same memory.
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();

    auto page_of = [&](int i) -> int { return i < count ? a.free_pages[count - 1 - i] : -1; };
    for (int b = me; b <= batch; b += stride) {
        a.cu_tokens[b] = cu[b];
        if (b < batch) {
            const int start = shift[b] + cu[b];
            a.start[b] = start;
            a.kv_len[b] = static_cast<int32_t>(min(static_cast<int64_t>(start) + (cu[b + 1] - cu[b]), static_cast<int64_t>(0x7fffffff)));
        }
    }
    for (int i = me; i < taken; i += stride) {
        const int b = last_at_or_below(pages, batch, i);
        a.block_table[b * a.table_stride + columns(shift[b] + cu[b]) + (i - pages[b])] = page_of(i);
    }
    // A token a thread, or four, most of them of one row and page: 9 rows of 7001 tokens 6.5 us, 7.9 with a row
    // and a look-up for each (with eight a thread 7.7).
    const int packed = cu[batch];
    const bool vec = aligned(a.positions, 16) && aligned(a.slots, 16);
    auto fill = [&](auto width) {
        constexpr int N = decltype(width)::value;
        auto store = [&](int64_t t0, const int (&pos)[N], const int (&slot)[N]) {
            if constexpr (N == 4) {
                if (vec && t0 + N <= total) {
                    *reinterpret_cast<int4 *>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                    *reinterpret_cast<int4 *>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                    return;
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (t0 + j < total) {
                    a.positions[t0 + j] = pos[j];
                    a.slots[t0 + j] = slot[j];
                }
        };
        for (int64_t t0 = N * static_cast<int64_t>(me); t0 < total; t0 += N * static_cast<int64_t>(stride)) {
            int pos[N], slot[N], b = t0 < packed ? last_at_or_below(cu, batch, static_cast<int>(t0)) : 0;
            if (N > 1 && ps >= N && t0 + N <= packed && t0 + N <= cu[b + 1] && shift[b] + t0 + N <= 0x7fffffff) {
                // tokens of one row, in two pages at most
                const int p0 = shift[b] + static_cast<int>(t0), col = static_cast<int>(page_in(p0)), off = p0 - col * static_cast<int>(ps);
                const int held = columns(shift[b] + cu[b]), first_new = pages[b];
                auto page_at = [&](int c) -> int {
                    if (c >= a.table_cols) return -1;
                    return c < held ? a.block_table[b * a.table_stride + c] : page_of(first_new + c - held);
                };
                const int page0 = page_at(col), page1 = off + N > static_cast<int>(ps) ? page_at(col + 1) : -1;
                const int64_t slot0 = static_cast<int64_t>(page0) * ps + off, slot1 = static_cast<int64_t>(page1) * ps + off - ps;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const bool in1 = off + j >= static_cast<int>(ps);
                    const int64_t s = (in1 ? slot1 : slot0) + j;
                    pos[j] = p0 + j;
                    slot[j] = (in1 ? page1 : page0) >= 0 && s <= 0x7fffffff ? static_cast<int>(s) : -1;
                }
                store(t0, pos, slot);
                continue;
            }
            const int32_t *from[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int64_t t = t0 + j;
                pos[j] = -1;
                from[j] = nullptr;  // where the token's page is found
                if (t >= packed) continue;
                while (cu[b + 1] <= t) ++b;
                pos[j] = static_cast<int>(min(static_cast<int64_t>(shift[b]) + t, static_cast<int64_t>(0x7fffffff)));
                if (pos[j] < reach) {
                    const int col = static_cast<int>(page_in(pos[j])), held = columns(shift[b] + cu[b]), i = pages[b] + col - held;
                    if (col < held) from[j] = a.block_table + b * a.table_stride + col;
                    else if (i < count) from[j] = a.free_pages + (count - 1 - i);
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) slot[j] = from[j] != nullptr ? *from[j] : -1;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int64_t s = static_cast<int64_t>(slot[j]) * ps + (pos[j] - static_cast<int64_t>(page_in(pos[j])) * ps);
                slot[j] = slot[j] >= 0 && s <= 0x7fffffff ? static_cast<int>(s) : -1;
            }
            store(t0, pos, slot);
        }
    };
    if (total <= stride) fill(std::integral_constant<int, 1>{});
    else fill(std::integral_constant<int, 4>{});
    if (me == 0) {
        *a.free_count_out = static_cast<int32_t>(max(count - taken, static_cast<int64_t>(0)));
        if (taken > count) record_device_error(err, kDevNoPages);
    }
}

}// namespace
}// namespace lcml

using namespace lcml;

extern "C" int lcml_kv_plan(const lcml_kv_plan_desc *d, lcml_stream_t stream) {
    LCML_CHECK_ARG(d != nullptr, "lcml_kv_plan: null descriptor");
    LCML_CHECK_ARG(d->batch >= 0 && d->batch <= kMaxRows, "lcml_kv_plan: batch %d is not in 0 .. %d", d->batch, kMaxRows);
    LCML_CHECK_ARG(d->page_size > 0 && d->page_size <= 65536, "lcml_kv_plan: page_size %d", d->page_size);
    LCML_CHECK_ARG(d->table_cols >= 0 && d->table_stride >= d->table_cols, "lcml_kv_plan: table_stride is less than table_cols, or negative");
    LCML_CHECK_ARG(d->total_tokens >= 0 && d->total_tokens <= 0x7fffffff, "lcml_kv_plan: total_tokens is not in 0 .. 2^31 - 1");
    // entries and columns are counted in 32 bits, by strides of up to kCluster * kThreads
    LCML_CHECK_ARG(static_cast<int64_t>(d->batch) * d->table_cols <= 0x7fffffff - 65536, "lcml_kv_plan: the table has over 2^31 - 65537 entries");
    LCML_CHECK_ARG(d->free_capacity >= 0, "lcml_kv_plan: negative free_capacity");
    LCML_CHECK_ARG(d->cu_tokens && d->free_count && d->free_count_out, "lcml_kv_plan: null pointer");
    LCML_CHECK_ARG(d->batch == 0 || (d->new_tokens && d->held && d->start && d->kv_len && (d->block_table || d->table_cols == 0)),
                   "lcml_kv_plan: null pointer");
    LCML_CHECK_ARG((d->total_tokens == 0 || (d->positions && d->slots)) && (d->free_capacity == 0 || d->free_pages), "lcml_kv_plan: null pointer");
    LCML_CHECK_ARG(aligned(d->block_table, 4) && aligned(d->new_tokens, 4) && aligned(d->held, 4) && aligned(d->free_pages, 4) && aligned(d->free_count, 4) &&
                       aligned(d->cu_tokens, 4) && aligned(d->start, 4) && aligned(d->kv_len, 4) && aligned(d->positions, 4) && aligned(d->slots, 4) &&
                       aligned(d->free_count_out, 4),
                   "lcml_kv_plan: a pointer is not 4-byte aligned");
    const int smem = (3 * d->batch + 2) * 4;
    const int rc = ensure_max_smem(reinterpret_cast<const void *>(k_kv_plan), (3 * kMaxRows + 2) * 4, "kv_plan");
    if (rc != LCML_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    // One CTA where it has a few rows and tokens a thread, else a cluster of 512 threads each (9 rows of
    // 7001 tokens: 6.5 us, with 256 threads 8.1, with 1024 7.0, as clusters of those start later), or of 1024
    // where more rows than warps may end (26 of 256 rows: 11.7 us, with 512 12.9).
    const int64_t work = d->batch > (d->total_tokens + 3) / 4 ? d->batch : (d->total_tokens + 3) / 4;
    const bool alone = work <= kThreads && d->ended == nullptr;
    cfg.gridDim = dim3(alone ? 1 : kCluster);
    cfg.blockDim = dim3(alone ? (work <= 128 ? 128 : static_cast<unsigned>((work + 31) / 32 * 32)) : (d->ended != nullptr && d->batch > kCluster * 16 ? kThreads : 512));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = to_cuda(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cfg.gridDim.x;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_kv_plan, *d, PageDivision(d->page_size), device_error_word());
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(LCML_ERR_CUDA, "kv_plan launch failed: %s", cudaGetErrorString(e));
    }
    return LCML_OK;
}
