// The paged key/value cache's bookkeeping: the page plan of a step (pages taken and
// given back, row offsets, positions and cache slots, all from lengths that live on
// the device) and the store of new key and value rows into their slots.
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
// that owned, top, table and the stack are updated in place between two block
// barriers without counters or a second read.  What bounds it is the launch and
// the chain lengths -> scan -> page -> slot, each an L2 round trip.  The rows are
// independent of one another: up to kPlanRows of them are done by the same CTA,
// more by a second launch over the whole GPU.
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
    bool bad;
};

__device__ __forceinline__ PlanRequest plan_request(const PlanArgs &a, int b) {
    PlanRequest r;
    r.context = a.context[b];
    r.count = a.count[b];
    r.owned = a.owned_in[b];
    const int64_t length = static_cast<int64_t>(r.context) + r.count;
    r.bad = r.context < 0 || r.count < 0 || length > (static_cast<int64_t>(a.table_width) << a.page_shift) ||
            r.owned < 0 || r.owned > a.table_width;
    if (r.bad) {
        r.context = r.count = 0;
        r.owned = r.need = r.owned < 0 ? 0 : (r.owned > a.table_width ? a.table_width : r.owned);
    } else {
        r.need = static_cast<int>((length + (1 << a.page_shift) - 1) >> a.page_shift);
    }
    return r;
}

// Inclusive scan of one value per thread over the block; `warp_sums` holds 32 values.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int64_t s = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += o;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    total = warp_sums[31];
    return v + (warp ? warp_sums[warp - 1] : 0);
}

// The last index i of ends[0 .. n) with (i ? ends[i - 1] : 0) <= x < ends[i].
template <typename T>
__device__ __forceinline__ int find_range(const T *ends, int n, T x) {
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

// Position and slot of token t of request b, which owns `held` pages, read from the
// finished table.  A token past them has no slot (its request was not served).
__device__ __forceinline__ void write_row(const PlanArgs &a, int64_t row, int b, int context, int t, int held) {
    const int position = context + t;
    int slot = -1;
    if ((position >> a.page_shift) < held) {
        const int page = a.table[b * a.table_ld + (position >> a.page_shift)];
        if (page >= 0 && page < a.pool)
            slot = (page << a.page_shift) + (position & ((1 << a.page_shift) - 1));
        else
            set_flag(a.flags, BD_FLAG_BAD_PAGE);
    }
    a.positions[row] = position;
    a.slots[row] = slot;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanArgs a) {
    __shared__ int64_t warp_sums[32];
    __shared__ int64_t ends[kPlanThreads];  // inclusive sums of a chunk of requests
    __shared__ int base[kPlanThreads];      // first table index given or taken by the request
    __shared__ int context[kPlanThreads], held[kPlanThreads];
    const int tid = threadIdx.x;
    grid_wait();
    grid_launch_dependents();
    int64_t top = a.top_in[0];
    if (top < 0 || top > a.free_capacity) {
        if (tid == 0) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        top = top < 0 ? 0 : a.free_capacity;
    }
    // pages given back go on top of the stack; the thread that moves one clears its entry
    int64_t given = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kPlanThreads) {
        const int b = b0 + tid;
        PlanRequest r{};
        if (b < a.requests) {
            r = plan_request(a, b);
            if (r.bad) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        }
        int64_t total;
        const int64_t end = block_scan(max(r.owned - r.need, 0), warp_sums, total);
        ends[tid] = end;
        base[tid] = r.need;
        __syncthreads();
        for (int64_t i = tid; i < total; i += kPlanThreads) {
            const int k = find_range(ends, kPlanThreads, i);
            const int64_t at = (b0 + k) * a.table_ld + base[k] + (i - (k ? ends[k - 1] : 0));
            const int page = a.table[at];
            a.table[at] = -1;
            if (top + given + i < a.free_capacity)
                a.free_list[top + given + i] = page;
            else
                set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        }
        given += total;
        __syncthreads();
    }
    const int64_t available = min(top + given, a.free_capacity);
    // pages taken come off it; a request whose pages do not all fit keeps what it has
    int64_t wanted = 0, taken = 0, row0 = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kPlanThreads) {
        const int b = b0 + tid;
        PlanRequest r{};
        if (b < a.requests) r = plan_request(a, b);
        const int lack = max(r.need - r.owned, 0);
        int64_t total, served_total;
        const int64_t end = wanted + block_scan(lack, warp_sums, total);
        const bool served = end <= available;
        if (lack && !served) set_flag(a.flags, BD_FLAG_NO_PAGES);
        // the served ones are the first: their sums are the places in the stack
        const int64_t mine = block_scan(served ? lack : 0, warp_sums, served_total);
        ends[tid] = mine;
        base[tid] = r.owned;
        context[tid] = r.context;
        held[tid] = lack && !served ? r.owned : r.need;
        __syncthreads();  // every thread of the chunk has read owned_in before owned_out (which may be the same)
        if (b < a.requests) a.owned_out[b] = held[tid];
        for (int64_t i = tid; i < served_total; i += kPlanThreads) {
            const int k = find_range(ends, kPlanThreads, i);
            int page = a.free_list[available - 1 - taken - i];
            if (page < 0 || page >= a.pool) {
                set_flag(a.flags, BD_FLAG_BAD_PAGE);
                page = -1;
            }
            a.table[(b0 + k) * a.table_ld + base[k] + (i - (k ? ends[k - 1] : 0))] = page;
        }
        wanted += total;
        taken += served_total;
        // row offsets of the chunk, and its rows
        int64_t rows_total;
        const int64_t row_end = block_scan(r.count, warp_sums, rows_total);
        ends[tid] = row_end;
        if (b < a.requests) a.starts[b] = static_cast<int>(row0 + row_end - r.count);
        __syncthreads();
        if (a.rows_here) {
            const int64_t live = min(rows_total, a.rows - row0);
            for (int64_t i = tid; i < live; i += kPlanThreads) {
                const int k = find_range(ends, kPlanThreads, i);
                write_row(a, row0 + i, b0 + k, context[k], static_cast<int>(i - (k ? ends[k - 1] : 0)), held[k]);
            }
        }
        row0 += rows_total;
        __syncthreads();
    }
    if (row0 > a.rows && tid == 0) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
    if (tid == 0) {
        a.starts[a.requests] = static_cast<int>(min(row0, static_cast<int64_t>(INT32_MAX)));
        a.top_out[0] = static_cast<int>(available - taken);
    }
    if (a.rows_here)
        for (int64_t i = row0 + tid; i < a.rows; i += kPlanThreads) a.positions[i] = a.slots[i] = -1;
}

// Positions and slots of many rows, once the plan's starts and table are written.
constexpr int kRowThreads = 256;
constexpr int kRowsEach = 4;

__global__ void __launch_bounds__(kRowThreads) page_rows_kernel(const PlanArgs a) {
    __shared__ int first;
    grid_wait();
    grid_launch_dependents();
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRowThreads * kRowsEach;
    const int64_t total = a.starts[a.requests];
    const int tid = threadIdx.x;
    // the request of the CTA's first row: a 32-way search by one warp
    if (tid < 32) {
        int lo = 0, n = a.requests;  // the answer is in [lo, lo + n)
        while (n > 1) {
            const int step = (n + 31) / 32;
            const int at = lo + tid * step;
            const bool below = at < lo + n && a.starts[at] <= r0;
            const unsigned vote = __ballot_sync(0xffffffffu, below);
            const int k = vote ? 31 - __clz(vote) : 0;
            lo += k * step;
            n = min(step, n - k * step);
        }
        if (tid == 0) first = lo;
    }
    __syncthreads();
    int b = first;
#pragma unroll
    for (int j = 0; j < kRowsEach; ++j) {
        const int64_t row = r0 + j * kRowThreads + tid;
        if (row >= a.rows) return;
        if (row >= total) {
            a.positions[row] = a.slots[row] = -1;
            continue;
        }
        // on from the thread's last request, in steps that double, then by halves
        int step = 1;
        while (b + step < a.requests && a.starts[b + step] <= row) {
            b += step;
            step <<= 1;
        }
        while (step > 1) {
            step >>= 1;
            if (b + step < a.requests && a.starts[b + step] <= row) b += step;
        }
        write_row(a, row, b, a.context[b], static_cast<int>(row - a.starts[b]), a.owned_out[b]);
    }
}

// ------------------------------------------------------------------ store
//
// One thread moves 8 values (16 bytes out) of a key or value row at a time and has
// kStoreEach such pieces in flight, which is what bounds it: HBM bytes in flight.
constexpr int kStoreThreads = 256;
constexpr int kStoreEach = 4;

struct StoreArgs {
    const void *k, *v;
    int64_t k_row, k_head, v_row, v_head;  // strides in elements
    const int32_t *slots;
    int64_t rows;
    int kv_heads, head_chunks;  // head_chunks = head_dim / 8
    int page_shift;
    int64_t pool;
    uint16_t *k_cache, *v_cache;
    CacheStrides ks, vs;
    int32_t *flags;
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
    const float4 lo = __ldg(reinterpret_cast<const float4 *>(p)), hi = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
    x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half *p, float (&x)[8]) {
    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

// Rounded to nearest even, the cache's one rounding; a value that is not finite
// afterwards (too large for the type, or not finite before) is reported.
template <bool BF16>
__device__ __forceinline__ uint32_t round_pair(float a, float b, bool &bad) {
    uint32_t u;
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        u = *reinterpret_cast<const uint32_t *>(&h);
        bad |= (u & 0x7F80u) == 0x7F80u || (u & 0x7F800000u) == 0x7F800000u;
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        u = *reinterpret_cast<const uint32_t *>(&h);
        bad |= (u & 0x7C00u) == 0x7C00u || (u & 0x7C000000u) == 0x7C000000u;
    }
    return u;
}

template <typename T, bool BF16>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const StoreArgs a) {
    grid_wait();
    grid_launch_dependents();
    const uint32_t chunks = static_cast<uint32_t>(a.kv_heads) * a.head_chunks;  // of one tensor's row
    const int64_t total = a.rows * 2 * chunks;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kStoreThreads * kStoreEach + threadIdx.x;
    float x[kStoreEach][8];
    int64_t to[kStoreEach];  // element offset in the cache, -1: nothing to store
    bool value[kStoreEach];
    bool bad_page = false, bad = false;
#pragma unroll
    for (int j = 0; j < kStoreEach; ++j) {
        const int64_t i = i0 + j * kStoreThreads;
        to[j] = -1;
        value[j] = false;
        if (i >= total) continue;
        const int64_t row = i / (2 * chunks);
        uint32_t c = static_cast<uint32_t>(i - row * (2 * chunks));
        value[j] = c >= chunks;
        c -= value[j] ? chunks : 0;
        const uint32_t head = c / a.head_chunks, at = (c - head * a.head_chunks) * 8;
        const int slot = __ldg(a.slots + row);
        if (slot < 0) continue;
        const int64_t page = slot >> a.page_shift;
        if (page >= a.pool) {
            bad_page = true;
            continue;
        }
        const CacheStrides &s = value[j] ? a.vs : a.ks;
        to[j] = page * s.page + (slot & ((1 << a.page_shift) - 1)) * s.slot + head * s.head + at;
        const T *src = value[j] ? static_cast<const T *>(a.v) + row * a.v_row + head * a.v_head
                                : static_cast<const T *>(a.k) + row * a.k_row + head * a.k_head;
        load8<T>(src + at, x[j]);
    }
#pragma unroll
    for (int j = 0; j < kStoreEach; ++j) {
        if (to[j] < 0) continue;
        uint4 w;
        w.x = round_pair<BF16>(x[j][0], x[j][1], bad);
        w.y = round_pair<BF16>(x[j][2], x[j][3], bad);
        w.z = round_pair<BF16>(x[j][4], x[j][5], bad);
        w.w = round_pair<BF16>(x[j][6], x[j][7], bad);
        *reinterpret_cast<uint4 *>((value[j] ? a.v_cache : a.k_cache) + to[j]) = w;
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
    int st = launch_pdl(page_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
    if (st || a.rows_here) return st;
    const unsigned grid = static_cast<unsigned>((rows + kRowThreads * kRowsEach - 1) / (kRowThreads * kRowsEach));
    return launch_pdl(page_rows_kernel, dim3(grid), dim3(kRowThreads), 0, stream, a);
}

template <typename T>
static int launch_store(const StoreArgs &a, bool bf16, cudaStream_t stream) {
    const int64_t pieces = a.rows * 2 * a.kv_heads * a.head_chunks;
    const int64_t grid = (pieces + kStoreThreads * kStoreEach - 1) / (kStoreThreads * kStoreEach);
    if (grid > INT32_MAX) return BD_ERR_TOO_LARGE;
    return launch_pdl(bf16 ? paged_store_kernel<T, true> : paged_store_kernel<T, false>,
                      dim3(static_cast<unsigned>(grid)), dim3(kStoreThreads), 0, stream, a);
}

extern "C" int bd_paged_store(const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head,
                              int row_type, const int32_t *slots, int64_t rows, int kv_heads, int head_dim,
                              int page_size, int64_t pool_pages, void *k_cache, const int64_t *k_strides,
                              void *v_cache, const int64_t *v_strides, int cache_type, int32_t *flags,
                              bd_stream_t stream) {
    if (rows < 0 || kv_heads < 1 || head_dim < 8 || head_dim % 8 || !page_size_ok(page_size) ||
        !pool_ok(pool_pages, page_size) || (row_type != BD_F32 && row_type != BD_F16 && row_type != BD_BF16) ||
        (cache_type != BD_F16 && cache_type != BD_BF16) || static_cast<int64_t>(kv_heads) * head_dim > (1 << 24))
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
    a.kv_heads = kv_heads;
    a.head_chunks = head_dim / 8;
    a.page_shift = log2_of(page_size);
    a.pool = pool_pages;
    a.k_cache = static_cast<uint16_t *>(k_cache);
    a.v_cache = static_cast<uint16_t *>(v_cache);
    a.flags = flags;
    const bool bf16 = cache_type == BD_BF16;
    if (row_type == BD_F32) return launch_store<float>(a, bf16, stream);
    if (row_type == BD_F16) return launch_store<__half>(a, bf16, stream);
    return launch_store<__nv_bfloat16>(a, bf16, stream);
}
