// The paged key/value cache's bookkeeping: the page plan of a step (pages taken and
// given back, row offsets, positions and cache slots, all from lengths that live on
// the device) and the store of new key and value rows into their slots.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "paged.cuh"

namespace bd {

// ------------------------------------------------------------------ page plan
//
// need_b = ceil((context_b + count_b) / page).  With G the pages that requests own
// beyond their need and K those they lack, the stack of free pages becomes
// S = free[0 .. top) ++ (pages given back, by request and table index), and the
// j-th lacking page, by request and table index, is S[top + G - 1 - j].
//
// One CTA does the scans over the requests and every table entry (a step changes
// few: a request of a draft round takes a page every page / accepted rounds), so
// that owned, top, table and the stack are updated in place between block barriers,
// without counters.  What bounds it is the launch and the chain lengths -> scan ->
// page -> slot, two L2 round trips: up to kPlanThreads requests are read once and
// scanned once, and a token on a page taken now reads the stack, not the table.
// 32 requests with 512 rows take 5.9 us, one request 3.1.
// The rows are independent of one another: up to kPlanRows of them are done by the
// same CTA, more by a second launch over the whole GPU (a CTA per request and
// stretch of tokens, so that no row looks its request up): 256 requests with 122,000 rows
// take 13.9 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 4096;

struct PlanArgs {
    const int32_t *context, *count, *owned_in;
    int32_t *owned_out;
    int requests, page_shift;
    int64_t pool;
    int32_t *table;
    int64_t table_ld;
    int table_width;
    int32_t *free_list;
    int64_t free_capacity;
    const int32_t *top_in;
    int32_t *top_out;
    int32_t *starts, *positions, *slots;
    int64_t rows;
    int rows_here;  // the plan kernel fills positions and slots itself
    int32_t *flags;
};

// A request as the plan sees it: bad lengths keep their pages and have no rows.
struct PlanRequest {
    int context, count, owned, need;
};

__device__ __forceinline__ PlanRequest plan_request(const PlanArgs &a, int b) {
    PlanRequest r{};
    if (b >= a.requests) return r;
    r.context = a.context[b];
    r.count = a.count[b];
    r.owned = a.owned_in[b];
    const int64_t length = static_cast<int64_t>(r.context) + r.count;
    if (r.context < 0 || r.count < 0 || length > (static_cast<int64_t>(a.table_width) << a.page_shift) || r.owned < 0 ||
        r.owned > a.table_width) {
        set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        r.context = r.count = 0;
        r.owned = r.need = r.owned < 0 ? 0 : (r.owned > a.table_width ? a.table_width : r.owned);
    } else {
        r.need = static_cast<int>((length + (1 << a.page_shift) - 1) >> a.page_shift);
    }
    return r;
}

// What is scanned over the requests: pages given back, pages lacking, rows.
struct PlanSums {
    int64_t give, lack, rows;
};

__device__ __forceinline__ PlanSums operator+(const PlanSums &x, const PlanSums &y) {
    return PlanSums{x.give + y.give, x.lack + y.lack, x.rows + y.rows};
}
__device__ __forceinline__ PlanSums plan_sums(const PlanRequest &r) {
    return PlanSums{max(r.owned - r.need, 0), max(r.need - r.owned, 0), r.count};
}

// Inclusive scan of one value per thread over the block; `warp_sums` holds 32 values.
__device__ __forceinline__ PlanSums block_scan(PlanSums v, PlanSums *warp_sums, PlanSums &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto warp_scan = [&](PlanSums x) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const PlanSums o{__shfl_up_sync(0xffffffffu, x.give, d), __shfl_up_sync(0xffffffffu, x.lack, d),
                             __shfl_up_sync(0xffffffffu, x.rows, d)};
            if (lane >= d) x = x + o;
        }
        return x;
    };
    v = warp_scan(v);
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) warp_sums[lane] = warp_scan(lane < (blockDim.x >> 5) ? warp_sums[lane] : PlanSums{0, 0, 0});
    __syncthreads();
    total = warp_sums[31];
    return warp ? v + warp_sums[warp - 1] : v;
}

// The first index i of the inclusive sums ends[0 .. n) with x < ends[i].
__device__ __forceinline__ int find_range(const int64_t *ends, int n, int64_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (x < ends[mid])
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ int checked_page(const PlanArgs &a, int page) {
    if (page >= 0 && page < a.pool) return page;
    set_flag(a.flags, BD_FLAG_BAD_PAGE);
    return -1;
}

__device__ __forceinline__ void write_row(const PlanArgs &a, int64_t row, int position, int page) {
    a.positions[row] = position;
    a.slots[row] = page < 0 ? -1 : (page << a.page_shift) + (position & ((1 << a.page_shift) - 1));
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanArgs a) {
    __shared__ PlanSums warp_sums[32];
    __shared__ int64_t give_end[kPlanThreads], lack_end[kPlanThreads], row_end[kPlanThreads];  // of a chunk of requests
    __shared__ PlanRequest chunk[kPlanThreads];
    __shared__ unsigned long long served_sum;
    const int tid = threadIdx.x, n = blockDim.x;
    grid_wait();
    grid_launch_dependents();
    const bool once = a.requests <= n;
    PlanRequest r = plan_request(a, tid);
    int64_t top = a.top_in[0];
    if (top < 0 || top > a.free_capacity) {
        if (tid == 0) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        top = top < 0 ? 0 : a.free_capacity;
    }
    if (tid == 0) served_sum = 0;
    PlanSums sums, total;
    // pages given back go on top of the stack; the thread that moves one clears its entry
    int64_t given = 0;
    for (int b0 = 0; b0 < a.requests; b0 += n) {
        if (b0) r = plan_request(a, b0 + tid);
        sums = block_scan(plan_sums(r), warp_sums, total);
        give_end[tid] = sums.give;
        lack_end[tid] = sums.lack;
        row_end[tid] = sums.rows;
        chunk[tid] = r;
        __syncthreads();
        for (int64_t i = tid; i < total.give; i += n) {
            const int k = find_range(give_end, n, i);
            const int64_t at = (b0 + k) * a.table_ld + chunk[k].need + (i - (k ? give_end[k - 1] : 0));
            const int page = a.table[at];
            checked_page(a, page);  // a bad one is reported by the step that gives it back too
            a.table[at] = -1;
            if (top + given + i < a.free_capacity)
                a.free_list[top + given + i] = page;
            else
                set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        }
        if (total.give) __syncthreads();
        given += total.give;
    }
    const int64_t available = min(top + given, a.free_capacity);
    // pages taken come off it; a request whose pages do not all fit keeps what it has.
    // The lacks add up in request order, so those that fit are the first ones.
    int64_t wanted = 0, row0 = 0;
    for (int b0 = 0; b0 < a.requests; b0 += n) {
        const int b = b0 + tid;
        if (!once) {
            r = plan_request(a, b);
            sums = block_scan(plan_sums(r), warp_sums, total);
            lack_end[tid] = sums.lack;
            row_end[tid] = sums.rows;
            chunk[tid] = r;
            __syncthreads();  // every thread of the chunk has read owned_in before owned_out (which may be the same)
        }
        const bool served = wanted + sums.lack <= available;
        if (r.need > r.owned && served)
            atomicMax(&served_sum, static_cast<unsigned long long>(wanted + sums.lack));
        else if (r.need > r.owned)
            set_flag(a.flags, BD_FLAG_NO_PAGES);
        if (b < a.requests) {
            a.owned_out[b] = served || r.need < r.owned ? r.need : r.owned;
            a.starts[b] = static_cast<int>(min(row0 + sums.rows - r.count, static_cast<int64_t>(INT32_MAX)));
        }
#pragma unroll 4
        for (int64_t i = tid; i < total.lack; i += n) {
            const int k = find_range(lack_end, n, i);
            if (wanted + lack_end[k] > available) break;
            a.table[(b0 + k) * a.table_ld + chunk[k].owned + (i - (k ? lack_end[k - 1] : 0))] =
                checked_page(a, a.free_list[available - 1 - wanted - i]);
        }
        if (a.rows_here) {
            const int64_t live = min(total.rows, a.rows - row0);
#pragma unroll 2
            for (int64_t i = tid; i < live; i += n) {
                const int k = find_range(row_end, n, i);
                const PlanRequest &q = chunk[k];
                const int position = q.context + static_cast<int>(i - (k ? row_end[k - 1] : 0));
                const int at = position >> a.page_shift;
                int page = -1;  // of a request that was not served
                if (at < q.owned)
                    page = checked_page(a, a.table[(b0 + k) * a.table_ld + at]);
                else if (wanted + lack_end[k] <= available)
                    page = checked_page(a, a.free_list[available - 1 - wanted - (k ? lack_end[k - 1] : 0) - (at - q.owned)]);
                write_row(a, row0 + i, position, page);
            }
        }
        wanted += total.lack;
        row0 += total.rows;
        __syncthreads();
    }
    if (tid == 0) {
        if (row0 > a.rows) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        a.starts[a.requests] = static_cast<int>(min(row0, static_cast<int64_t>(INT32_MAX)));
        a.top_out[0] = static_cast<int>(available - static_cast<int64_t>(served_sum));
    }
    if (a.rows_here)
        for (int64_t i = row0 + tid; i < a.rows; i += n) a.positions[i] = a.slots[i] = -1;
}

// Positions and slots of many rows, once the plan's starts and table are written: CTA
// (b, y) has every gridDim.y-th stretch of 256 tokens of request b; the last b has the
// rows behind the requests.
constexpr int kRowThreads = 256;

__global__ void __launch_bounds__(kRowThreads) page_rows_kernel(const PlanArgs a) {
    grid_wait();
    grid_launch_dependents();
    const int b = blockIdx.x;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * kRowThreads + threadIdx.x, step = gridDim.y * kRowThreads;
    const int64_t start = a.starts[b];
    if (b == a.requests) {
        for (int64_t row = start + first; row < a.rows; row += step) a.positions[row] = a.slots[row] = -1;
        return;
    }
    const int64_t end = min(static_cast<int64_t>(a.starts[b + 1]), a.rows);
    const int context = a.context[b], owned = a.owned_out[b];
    for (int64_t row = start + first; row < end; row += step) {
        const int position = context + static_cast<int>(row - start), at = position >> a.page_shift;
        write_row(a, row, position, at < owned ? checked_page(a, a.table[b * a.table_ld + at]) : -1);
    }
}

// ------------------------------------------------------------------ store
//
// A thread moves one piece of 8 values (16 bytes out), always the same one of a row, of
// kStoreEach rows at a time: with nothing to divide per piece and all its loads in
// flight, what bounds it is HBM: 30,000 bf16 rows of 2 x 2 KB take 39.1 us = 6.3 TB/s, 6,200
// fp32 rows of 2 x 1.25 KB into bf16 4.1 us = 5.8 TB/s, 512 rows 2.6 us.
constexpr int kStoreThreads = 256;
constexpr int kStoreEach = 4;

struct StoreArgs {
    const void *k, *v;
    int64_t k_row, k_head, v_row, v_head;  // strides in elements
    const int32_t *slots;
    int64_t rows;
    int head_chunks, chunks;  // pieces of a head, and of a row of one tensor
    int rows_each;            // rows that a CTA passes over at once
    int page_shift;
    int64_t pool;
    uint16_t *k_cache, *v_cache;
    CacheStrides ks, vs;
    int32_t *flags;
};

// Rounded to nearest even, the cache's one rounding.
template <bool BF16>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// A value too large for the type, or not finite before.
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t u) {
    constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
    return (u & e) == e || (u & (e << 16)) == (e << 16);
}

// 8 values as they are loaded (T: float, __half, __nv_bfloat16) and as they are stored.
template <typename T>
struct Piece {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ float2 pair(int i) const {
        if (sizeof(T) == 4) {
            const uint4 &x = w[i >> 1 < static_cast<int>(sizeof(T) / 2) ? i >> 1 : 0];
            return (i & 1) ? make_float2(__uint_as_float(x.z), __uint_as_float(x.w))
                           : make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
        }
        const uint32_t u = i == 0 ? w[0].x : (i == 1 ? w[0].y : (i == 2 ? w[0].z : w[0].w));
        if (std::is_same<T, __nv_bfloat16>::value)
            return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
        return __half22float2(*reinterpret_cast<const __half2 *>(&u));
    }
    template <bool BF16>
    __device__ __forceinline__ uint4 rounded() const {
        if (std::is_same<T, typename std::conditional<BF16, __nv_bfloat16, __half>::type>::value) return w[0];
        const float2 a = pair(0), b = pair(1), c = pair(2), d = pair(3);
        return make_uint4(round_pair<BF16>(a.x, a.y), round_pair<BF16>(b.x, b.y), round_pair<BF16>(c.x, c.y),
                          round_pair<BF16>(d.x, d.y));
    }
};

template <typename T, bool BF16>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const StoreArgs a) {
    grid_wait();
    grid_launch_dependents();
    // the piece: of a row if the CTA holds whole rows, else of the blockIdx.y-th part of one
    const int pieces = 2 * a.chunks;
    const int lane_row = a.rows_each > 1 ? threadIdx.x / pieces : 0;
    int c = a.rows_each > 1 ? threadIdx.x - lane_row * pieces : blockIdx.y * kStoreThreads + threadIdx.x;
    if (lane_row >= a.rows_each || c >= pieces) return;
    const bool value = c >= a.chunks;
    c -= value ? a.chunks : 0;
    const int head = c / a.head_chunks, at = (c - head * a.head_chunks) * 8;
    const CacheStrides s = value ? a.vs : a.ks;
    const int64_t row_stride = value ? a.v_row : a.k_row;
    const T *src = static_cast<const T *>(value ? a.v : a.k) + head * (value ? a.v_head : a.k_head) + at;
    uint16_t *dst = (value ? a.v_cache : a.k_cache) + head * s.head + at;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.rows_each * kStoreEach + lane_row;
    Piece<T> x[kStoreEach];
    int slot[kStoreEach];
    bool bad_page = false, bad = false;
#pragma unroll
    for (int j = 0; j < kStoreEach; ++j) {
        const int64_t row = row0 + j * a.rows_each;
        slot[j] = row < a.rows ? a.slots[row] : -1;
        x[j].load(src + min(row, a.rows - 1) * row_stride);
    }
#pragma unroll
    for (int j = 0; j < kStoreEach; ++j) {
        if (slot[j] < 0) continue;
        const int64_t page = slot[j] >> a.page_shift;
        if (page >= a.pool) {
            bad_page = true;
            continue;
        }
        const uint4 w = x[j].template rounded<BF16>();
        bad |= not_finite<BF16>(w.x) || not_finite<BF16>(w.y) || not_finite<BF16>(w.z) || not_finite<BF16>(w.w);
        *reinterpret_cast<uint4 *>(dst + page * s.page + (slot[j] & ((1 << a.page_shift) - 1)) * s.slot) = w;
    }
    if (bad) set_flag(a.flags, BD_FLAG_CACHE_OVERFLOW);
    if (bad_page) set_flag(a.flags, BD_FLAG_BAD_PAGE);
}

}  // namespace bd

using namespace bd;

extern "C" int bd_page_plan(const int32_t *context, const int32_t *count, int requests, int page_size,
                            int64_t pool_pages, int32_t *table, int64_t table_ld, int table_width,
                            const int32_t *owned_in, int32_t *owned_out, int32_t *free_list, int64_t free_capacity,
                            const int32_t *top_in, int32_t *top_out, int32_t *starts, int32_t *positions,
                            int32_t *slots, int64_t rows, int32_t *flags, bd_stream_t stream) {
    if (requests < 1 || !page_size_ok(page_size) || !pool_ok(pool_pages, page_size) || table_width < 1 ||
        table_ld < table_width || !table_ok(table_width, page_size) || free_capacity < 0 || free_capacity > INT32_MAX ||
        rows < 0 || rows > INT32_MAX || !context || !count || !table || !owned_in || !owned_out || !top_in || !top_out ||
        !starts || (free_capacity && !free_list) || (rows && (!positions || !slots)))
        return BD_ERR_INVALID;
    PlanArgs a{};
    a.context = context;
    a.count = count;
    a.owned_in = owned_in;
    a.owned_out = owned_out;
    a.requests = requests;
    a.page_shift = log2_of(page_size);
    a.pool = pool_pages;
    a.table = table;
    a.table_ld = table_ld;
    a.table_width = table_width;
    a.free_list = free_list;
    a.free_capacity = free_capacity;
    a.top_in = top_in;
    a.top_out = top_out;
    a.starts = starts;
    a.positions = positions;
    a.slots = slots;
    a.rows = rows;
    a.rows_here = rows <= kPlanRows;
    a.flags = flags;
    // Barriers and scans are shorter with fewer warps, rows want a thread each: 32 requests
    // with 512 rows take 6.6 us with 256 threads, 5.9 us with 512.
    const int threads = requests <= 256 && rows <= 256   ? 256
                        : requests <= 512 && rows <= 1024 ? 512
                                                          : kPlanThreads;
    int st = launch_pdl(page_plan_kernel, dim3(1), dim3(threads), 0, stream, a);
    if (st || a.rows_here) return st;
    // twice the stretches of an average request, so that longer ones spread too
    const int64_t stretches = std::min<int64_t>(64, 2 * (rows / requests / kRowThreads + 1));
    return launch_pdl(page_rows_kernel, dim3(requests + 1, static_cast<unsigned>(stretches)), dim3(kRowThreads), 0, stream, a);
}

template <typename T>
static int launch_store(const StoreArgs &a, bool bf16, cudaStream_t stream) {
    const int64_t pass = static_cast<int64_t>(a.rows_each) * kStoreEach;
    const dim3 grid(static_cast<unsigned>((a.rows + pass - 1) / pass),
                    static_cast<unsigned>(a.rows_each > 1 ? 1 : (2 * a.chunks + kStoreThreads - 1) / kStoreThreads));
    return launch_pdl(bf16 ? paged_store_kernel<T, true> : paged_store_kernel<T, false>, grid, dim3(kStoreThreads), 0,
                      stream, a);
}

// No two (page, slot, head) of a cache share an element: each stride is beyond all that the
// smaller ones reach.
static bool apart(const CacheStrides &s, int64_t pages, int page_size, int heads, int head_dim) {
    std::pair<int64_t, int64_t> axes[3] = {{s.page, pages}, {s.slot, page_size}, {s.head, heads}};  // stride, size
    std::sort(axes, axes + 3);
    int64_t reach = head_dim;
    for (auto &axis : axes) {
        if (axis.second < 2) continue;
        if (axis.first < reach) return false;
        reach += (axis.second - 1) * axis.first;
    }
    return true;
}

extern "C" int bd_paged_store(const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head,
                              int row_type, const int32_t *slots, int64_t rows, int kv_heads, int head_dim,
                              int page_size, int64_t pool_pages, void *k_cache, const int64_t *k_strides,
                              void *v_cache, const int64_t *v_strides, int cache_type, int32_t *flags,
                              bd_stream_t stream) {
    if (rows < 0 || rows > INT32_MAX || kv_heads < 1 || head_dim < 8 || head_dim % 8 || !page_size_ok(page_size) ||
        !pool_ok(pool_pages, page_size) || (row_type != BD_F32 && row_type != BD_F16 && row_type != BD_BF16) ||
        (cache_type != BD_F16 && cache_type != BD_BF16) || static_cast<int64_t>(kv_heads) * head_dim > (1 << 20))
        return BD_ERR_INVALID;
    if (rows == 0) return BD_OK;
    if (!k || !v || !slots || !k_cache || !v_cache || !k_strides || !v_strides) return BD_ERR_INVALID;
    const int64_t unit = row_type == BD_F32 ? 4 : 8;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) ||
        ((k_row | k_head | v_row | v_head) % unit) != 0)
        return BD_ERR_ALIGNMENT;
    StoreArgs a{};
    if (!cache_strides(k_strides, a.ks) || !cache_strides(v_strides, a.vs)) return BD_ERR_ALIGNMENT;
    a.k = k;
    a.v = v;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    a.slots = slots;
    a.rows = rows;
    a.head_chunks = head_dim / 8;
    a.chunks = kv_heads * a.head_chunks;
    a.rows_each = std::max(1, kStoreThreads / (2 * a.chunks));
    a.page_shift = log2_of(page_size);
    a.pool = pool_pages;
    a.k_cache = static_cast<uint16_t *>(k_cache);
    a.v_cache = static_cast<uint16_t *>(v_cache);
    a.flags = flags;
    // slots that share elements would be written in any order
    if (!apart(a.ks, pool_pages, page_size, kv_heads, head_dim) || !apart(a.vs, pool_pages, page_size, kv_heads, head_dim) ||
        span_of(k_cache, 2 * head_dim).meets(span_of(v_cache, 2 * head_dim)))
        return BD_ERR_INVALID;
    const bool bf16 = cache_type == BD_BF16;
    if (row_type == BD_F32) return launch_store<float>(a, bf16, stream);
    if (row_type == BD_F16) return launch_store<__half>(a, bf16, stream);
    return launch_store<__nv_bfloat16>(a, bf16, stream);
}
