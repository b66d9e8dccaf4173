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
// Bound: latency. A step of 64 rows moves 2 KB.
#include "lcml_decoder.cuh"

#include "../../include/lcml_decode_step.h"

namespace lcml {
namespace {

constexpr int kDevNoPages = 8;  // joins the codes of DeviceError: the free list ran out
constexpr int kMaxRows = 16384;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;

__device__ __forceinline__ int64_t add_up(int64_t v, int lane) {  // inclusive sums of a warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// Exclusive sums of one value a thread over the block; `total` gets the block's.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t incl = add_up(v, lane);
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    const int64_t of = lane < (blockDim.x >> 5) ? warp_sums[lane] : 0;
    const int64_t upto = add_up(of, lane);
    total = __shfl_sync(0xffffffffu, upto, 31);
    const int64_t before = __shfl_sync(0xffffffffu, upto - of, warp);
    __syncthreads();
    return before + incl - v;
}

// The last i in [0, n) with first[i] <= x; first[0] <= x, not decreasing.
__device__ __forceinline__ int last_at_or_below(const int32_t *first, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) k_kv_plan(lcml_kv_plan_desc a, int *err) {
    extern __shared__ int32_t smem[];
    __shared__ int64_t warp_sums[kWarps];
    const int batch = a.batch;
    int32_t *cu = smem;                    // [batch + 1]
    int32_t *shift = smem + batch + 1;     // [batch]: a token's position less its packed index
    int32_t *pages = shift + batch;        // [batch + 1]: new entries of the rows before; at first, pages given back
    const int lane = threadIdx.x & 31;
    const int ctas = gridDim.x, rank = blockIdx.x;
    const int stride = ctas * blockDim.x, me = rank * blockDim.x + threadIdx.x;
    const int ps = a.page_size;
    const int64_t reach = static_cast<int64_t>(a.table_cols) * ps;
    bool bad = false;

    griddep_launch_dependents();
    griddep_wait();
    const int listed = *a.free_count;
    const int64_t capacity = a.free_capacity < 0x7fffffff ? a.free_capacity : 0x7fffffff;
    int64_t count = listed < 0 ? 0 : (listed < capacity ? listed : capacity);
    bad |= count != listed;

    auto columns = [&](int64_t tokens) -> int {  // columns of the table that hold this many
        return static_cast<int>(tokens < reach ? (tokens + ps - 1) / ps : a.table_cols);
    };
    if (a.ended != nullptr) {
        // a warp per row, the rows dealt to the cluster's warps; a count goes to every CTA
        auto row_entry = [&](int b, int c, int n) -> int { return c < n ? a.block_table[b * a.table_stride + c] : -1; };
        const int warps = stride >> 5, w = me >> 5;
        cluster_sync_all();  // every CTA has started
        for (int b = w; b < batch; b += warps) {
            int n = 0;
            if (a.ended[b] != 0) {
                const int cols = columns(max(0, a.held[b]));
                for (int c0 = 0; c0 < cols; c0 += 32) n += __popc(__ballot_sync(0xffffffffu, row_entry(b, c0 + lane, cols) >= 0));
            }
            if (lane < ctas) {
                const uint32_t to = mapa_shared(smem_u32(pages + b), lane);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(n) : "memory");
            }
        }
        cluster_sync_all();
        int64_t back = 0;
        for (int b0 = 0; b0 < batch; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            int64_t sum;
            const int64_t before = block_scan(b < batch ? pages[b] : 0, warp_sums, sum);
            if (b < batch) pages[b] = static_cast<int32_t>(back + before);
            back += sum;
        }
        __syncthreads();
        for (int b = w; b < batch; b += warps) {
            if (a.ended[b] == 0) continue;
            const int cols = columns(max(0, a.held[b]));
            int64_t at = count + pages[b];
            for (int c0 = 0; c0 < cols; c0 += 32) {
                const int p = row_entry(b, c0 + lane, cols);
                const uint32_t have = __ballot_sync(0xffffffffu, p >= 0);
                const int64_t to = at + __popc(have & ((1u << lane) - 1));
                if (p >= 0) {
                    if (to < capacity) a.free_pages[to] = p;
                    a.block_table[b * a.table_stride + c0 + lane] = -1;
                }
                at += __popc(have);
            }
        }
        bad |= count + back > capacity;
        count = count + back < capacity ? count + back : capacity;
        cluster_sync_all();  // the free list is complete, and `pages` may be written again
    }

    // sums of the tokens and of the new entries
    int64_t tokens = 0, taken = 0;
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
        int64_t sum;
        const int64_t first = tokens + block_scan(n, warp_sums, sum);
        tokens += sum;
        const int from = static_cast<int>(min(first, a.total_tokens)), to = static_cast<int>(min(first + n, a.total_tokens));
        const int64_t len = min(static_cast<int64_t>(start) + (to - from), static_cast<int64_t>(0x7fffffff));
        bad |= b < batch && (len > reach || to - from < n);
        const int64_t entries = taken + block_scan(b < batch ? columns(len) - columns(start) : 0, warp_sums, sum);
        taken += sum;
        if (b < batch) {
            cu[b] = from;
            shift[b] = start - from;
            pages[b] = static_cast<int32_t>(entries);
        }
    }
    if (threadIdx.x == 0) {
        cu[batch] = static_cast<int32_t>(min(tokens, a.total_tokens));
        pages[batch] = static_cast<int32_t>(taken);
    }
    if (rank == 0 && bad) record_device_error(err, kDevBadBatch);
    cluster_sync_all();  // every CTA has read held and free_count: kv_len and free_count_out may be the same memory

    auto page_of = [&](int64_t i) -> int { return i < count ? a.free_pages[count - 1 - i] : -1; };
    for (int b = me; b <= batch; b += stride) {
        a.cu_tokens[b] = cu[b];
        if (b < batch) {
            const int64_t start = static_cast<int64_t>(shift[b]) + cu[b];
            a.start[b] = static_cast<int32_t>(start);
            a.kv_len[b] = static_cast<int32_t>(min(start + (cu[b + 1] - cu[b]), static_cast<int64_t>(0x7fffffff)));
        }
    }
    for (int64_t i = me; i < taken; i += stride) {
        const int b = last_at_or_below(pages, batch, static_cast<int>(i));
        const int col = columns(static_cast<int64_t>(shift[b]) + cu[b]) + static_cast<int>(i - pages[b]);
        a.block_table[b * a.table_stride + col] = page_of(i);
    }
    const int packed = cu[batch];
    for (int64_t t = me; t < a.total_tokens; t += stride) {
        int pos = -1, slot = -1;
        if (t < packed) {
            const int b = last_at_or_below(cu, batch, static_cast<int>(t));
            pos = static_cast<int>(min(static_cast<int64_t>(shift[b]) + t, static_cast<int64_t>(0x7fffffff)));
            const int col = pos / ps;
            if (pos < reach) {
                const int held = columns(static_cast<int64_t>(shift[b]) + cu[b]);
                const int page = col < held ? a.block_table[b * a.table_stride + col] : page_of(static_cast<int64_t>(pages[b]) + col - held);
                const int64_t s = static_cast<int64_t>(page) * ps + (pos - col * ps);
                slot = page >= 0 && s <= 0x7fffffff ? static_cast<int>(s) : -1;
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
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
    LCML_CHECK_ARG(static_cast<int64_t>(d->batch) * d->table_cols <= 0x7fffffff, "lcml_kv_plan: the table has over 2^31 - 1 entries");
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
    cfg.gridDim = dim3(kCluster);
    cfg.blockDim = dim3(kThreads);
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_kv_plan, *d, device_error_word());
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(LCML_ERR_CUDA, "kv_plan launch failed: %s", cudaGetErrorString(e));
    }
    return LCML_OK;
}
