// Work split and row helpers of the paged attention, shared by its kernels.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace bd {

enum PagedMode : int {
    PAGED_F32 = 0,   // fp32 rows over an fp16 cache
    PAGED_F16 = 1,   // fp16 rows and cache
    PAGED_BF16 = 2,  // bf16 rows and cache
};

struct PagedOpen;

struct PagedArgs {
    const void *q;
    int64_t q_row, q_head;  // strides in elements
    const uint16_t *k, *v;
    CacheStrides ks, vs;
    const int32_t *table;
    int64_t table_ld;
    int table_width;
    int64_t pool;
    const int32_t *context, *starts;
    int requests;
    int64_t rows;  // rows of q and out
    int kv_heads, groups, page_shift;
    uint32_t group_mul, group_shift;  // row / groups, see paged_token()
    int causal, window, longest;  // window 0: none
    float scale_log2;             // scale x log2 e
    void *out;
    int64_t out_row;  // heads stand head_dim apart
    int zero_fill;
    int item_rows;   // rows of an item of the mma.sync kernel
    int split_rows;  // requests of more rows per kv head go to the tcgen05 kernel (INT_MAX: none, 0: all)
    // partials of the two kernels: [2 x CTAs][rows of an item][head_dim] and [..][2], and what to join
    struct Parts {
        float *o, *ml;
        PagedOpen *open;  // [CTAs]
    } parts[2];
    int32_t *flags;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// An output lies between the values that it weights, so fp16 ones are at most 65504, which the
// roundings of the weights can pass by 2^-11.  (Rows that are not finite are done again.)
template <int MODE>
__device__ __forceinline__ float paged_bounded(float x) {
    return MODE == PAGED_F16 ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
}

// row / groups for 0 <= row < 2^31: with 2^(s-1) < groups <= 2^s and the multiplier
// m = ceil(2^(31+s) / groups) < 2^32, row m 2^-(31+s) exceeds row / groups by less than
// row 2^-(31+s) < 1 / groups, so the floors agree.
__device__ __forceinline__ int paged_token(const PagedArgs &a, int row) {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.group_mul) >> a.group_shift);
}
inline void paged_set_groups(PagedArgs &a, int groups) {
    int s = 0;
    while ((1 << s) < groups) ++s;
    a.groups = groups;
    a.group_shift = 31 + s;
    a.group_mul = static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + groups - 1) / groups);
}

// A request's lengths; one whose lengths do not fit has no tokens.
struct PagedRequest {
    int row0, count, context;
    bool bad;
};

__device__ __forceinline__ PagedRequest paged_request(const PagedArgs &a, int b) {
    PagedRequest r;
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    r.context = a.context[b];
    r.row0 = s0;
    const int64_t count = static_cast<int64_t>(s1) - s0;
    r.bad = s0 < 0 || count < 0 || s1 > a.rows || r.context < 0 || count > a.longest ||
            r.context + count > (static_cast<int64_t>(a.table_width) << a.page_shift);
    r.count = r.bad ? 0 : static_cast<int>(count);
    return r;
}

// Keys [lo, hi) that token t of a request sees.
__device__ __forceinline__ void paged_token_range(const PagedArgs &a, int context, int count, int t, int &lo, int &hi) {
    const int p = context + t;
    hi = a.causal ? p + 1 : context + count;
    lo = 0;
    if (a.window) {
        lo = max(0, p - a.window + 1);
        if (a.window < hi - p) hi = p + a.window;
    }
}

// Rows [r0, r1) (token x groups + head of the group) of one request and kv head.
struct PagedItem {
    int b, h, r0, r1;
    int row0, count, context;
    int lo, hi;          // keys that some row sees
    int lo_all, hi_all;  // keys that every row sees
};

template <int M>
__device__ __forceinline__ void paged_item(const PagedArgs &a, const PagedRequest &r, int i, PagedItem &it) {
    it.row0 = r.row0;
    it.count = r.count;
    it.context = r.context;
    it.r0 = i * M;
    it.r1 = min(it.r0 + M, r.count * a.groups);
    paged_token_range(a, r.context, r.count, paged_token(a, it.r0), it.lo, it.hi_all);
    paged_token_range(a, r.context, r.count, paged_token(a, it.r1 - 1), it.lo_all, it.hi);
}

__device__ __forceinline__ void paged_row_range(const PagedArgs &a, const PagedItem &it, int row, int &lo, int &hi) {
    if (row < it.r1) {
        paged_token_range(a, it.context, it.count, paged_token(a, row), lo, hi);
    } else {
        lo = hi = 0;
    }
}

// Element offset of a row in a tensor of the given token and head strides.
__device__ __forceinline__ int64_t paged_row_offset(const PagedArgs &a, const PagedItem &it, int row, int64_t token_stride,
                                                    int64_t head_stride) {
    const int t = paged_token(a, row);
    return (static_cast<int64_t>(it.row0) + t) * token_stride +
           (static_cast<int64_t>(it.h) * a.groups + (row - t * a.groups)) * head_stride;
}

// An item that a CTA begins and does not end: its partials are place 2 c + 1 of this
// CTA c and places 2 d of the CTAs d = c + 1 .. last.
struct PagedOpen {
    PagedItem it;
    int last;  // -1: no such item
};

struct PagedShared {
    int64_t warp_sums[32];
    int64_t before, each;
    int b;
};

// The walk over this CTA's range of the batch, see the head of paged_attention.cu: the
// items of M rows and units of KT keys of the requests of one kernel (TC: those of
// more than a.split_rows rows per kv head, else the others).  An item counts as its
// units and EXTRA more, which is what a stay costs beside its tiles; a range that
// ends within these leaves the item to the next CTA.
template <int M, int KT, int EXTRA, bool TC>
struct PagedWalk {
    int cta, len, per;          // this CTA's range, and that of every CTA but the last
    int at;                     // where the current item begins, counted from the range's begin (first: <= 0)
    int b, h, i, tiles, units;  // units: of the item
    PagedRequest r;

    static __device__ __forceinline__ int item_units(const PagedItem &x) { return (x.hi + KT - 1) / KT - x.lo / KT; }
    static __device__ __forceinline__ int request_tiles(const PagedArgs &a, const PagedRequest &r) {
        const int rows = r.count * a.groups;
        return (rows > a.split_rows) == TC ? (rows + M - 1) / M : 0;
    }
    static __device__ __forceinline__ int cost(const PagedArgs &a, const PagedRequest &r, int i) {
        PagedItem x;
        paged_item<M>(a, r, i, x);
        return item_units(x) + EXTRA;
    }

    // Cost of one kv head of request b, a request to a lane; those of many items by the whole warp.
    static __device__ __forceinline__ int64_t request_cost(const PagedArgs &a, int b, PagedRequest &r) {
        r = PagedRequest{};
        if (b < a.requests) {
            r = paged_request(a, b);
            if (r.bad) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        }
        const int tiles = b < a.requests ? request_tiles(a, r) : 0;
        int64_t sum = 0;
        if (tiles <= 4)
            for (int i = 0; i < tiles; ++i) sum += cost(a, r, i);
        const int lane = threadIdx.x & 31;
        for (unsigned many = __ballot_sync(0xffffffffu, tiles > 4); many; many &= many - 1) {
            const int src = __ffs(many) - 1;
            PagedRequest q{};
            q.count = __shfl_sync(0xffffffffu, r.count, src);
            q.context = __shfl_sync(0xffffffffu, r.context, src);
            const int n = __shfl_sync(0xffffffffu, tiles, src);
            int64_t part = 0;
            for (int i = lane; i < n; i += 32) part += cost(a, q, i);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
            if (lane == src) sum = part;
        }
        return sum;
    }

    // Inclusive sum over the block, and its total.
    static __device__ __forceinline__ int64_t scan(int64_t v, PagedShared &sh, int64_t &sum) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += o;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sums[warp] = v;
        __syncthreads();
        int64_t before = 0;
        sum = 0;
        for (int w = 0; w < warps; ++w) {
            if (w == warp) before = sum;
            sum += sh.warp_sums[w];
        }
        return v + before;
    }

    __device__ __forceinline__ void set_request(const PagedArgs &a) {
        r = paged_request(a, b);
        tiles = request_tiles(a, r);
    }

    // Dividing 64-bit values takes some 300 cycles at a CTA's begin.
    static __device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
        return (x | y) >> 32 ? x / y : static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y));
    }

    // This CTA's range [u, u + len) of `ctas` equal ones of `total`; false when it is empty.
    __device__ __forceinline__ bool range(int64_t total, int ctas, int64_t &u) {
        per = static_cast<int>(divide(total + ctas - 1, ctas));
        u = static_cast<int64_t>(cta) * per;
        len = static_cast<int>(min(static_cast<int64_t>(per), total - u));
        return u < total;
    }

    // Places the walk at the begin of this CTA's range; false when it is empty.
    __device__ __forceinline__ bool begin(const PagedArgs &a, PagedShared &sh, int cta_, int ctas) {
        cta = cta_;
        const int n = blockDim.x, tid = threadIdx.x, lane = tid & 31;
        int64_t total, u, each, rest;  // each: cost of one kv head of the request around u
        if (a.requests <= 32) {  // every warp for itself, without a barrier
            PagedRequest mine;
            const int64_t cost = request_cost(a, lane, mine);
            int64_t incl = cost * a.kv_heads;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            total = __shfl_sync(0xffffffffu, incl, 31);
            if (!range(total, ctas, u)) return false;
            b = __ffs(__ballot_sync(0xffffffffu, u < incl)) - 1;
            each = __shfl_sync(0xffffffffu, cost, b);
            rest = u - (__shfl_sync(0xffffffffu, incl, b) - each * a.kv_heads);
            r.row0 = __shfl_sync(0xffffffffu, mine.row0, b);
            r.count = __shfl_sync(0xffffffffu, mine.count, b);
            r.context = __shfl_sync(0xffffffffu, mine.context, b);
            r.bad = false;  // it has rows
            tiles = request_tiles(a, r);
        } else {
            PagedRequest unused;
            int64_t sum, cost = request_cost(a, tid, unused);
            int64_t incl = scan(cost * a.kv_heads, sh, total);
            for (int b0 = n; b0 < a.requests; b0 += n) {
                scan(request_cost(a, b0 + tid, unused) * a.kv_heads, sh, sum);
                total += sum;
            }
            if (!range(total, ctas, u)) return false;
            int64_t before = 0;
            sum = total;
            for (int b0 = 0; b0 < a.requests; b0 += n) {
                if (a.requests > n) {
                    cost = request_cost(a, b0 + tid, unused);
                    incl = scan(cost * a.kv_heads, sh, sum);
                }
                if (before + incl - cost * a.kv_heads <= u && u < before + incl) {
                    sh.b = b0 + tid;
                    sh.before = before + incl - cost * a.kv_heads;
                    sh.each = cost;
                }
                before += sum;
                if (u < before) break;
            }
            __syncthreads();
            b = sh.b;
            each = sh.each;
            rest = u - sh.before;
            set_request(a);
        }
        // its kv head, and the item: 32 at a time, every warp for itself
        h = static_cast<int>(divide(rest, each));
        rest -= h * each;
        for (int i0 = 0;; i0 += 32) {
            const int mine = i0 + lane < tiles ? cost(a, r, i0 + lane) : 0;
            int end = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, end, d);
                if (lane >= d) end += o;
            }
            const unsigned found = __ballot_sync(0xffffffffu, rest < end);
            if (found) {
                const int src = __ffs(found) - 1;
                i = i0 + src;
                at = -static_cast<int>(rest - __shfl_sync(0xffffffffu, end - mine, src));
                break;
            }
            rest -= __shfl_sync(0xffffffffu, end, 31);
            if (i0 + 32 >= tiles) return false;  // not reached: the request holds u
        }
        return true;
    }

    // The next stay: an item, its key tiles [kt0, kt1), and the place of the partial it
    // leaves (-1: it is done whole).  An odd place is an item that later CTAs end.
    // False at the end of the range.
    __device__ __forceinline__ bool next(const PagedArgs &a, PagedItem &it, int &kt0, int &kt1, int &part) {
        while (at < len) {
            if (i == tiles) {
                i = 0;
                if (++h == a.kv_heads) {
                    h = 0;
                    do {
                        ++b;
                        set_request(a);
                    } while (tiles == 0);
                }
            }
            paged_item<M>(a, r, i, it);
            it.b = b;
            it.h = h;
            units = item_units(it);
            const int first = max(0, -at - EXTRA), last = min(units, len - at - EXTRA);
            at += units + EXTRA;
            ++i;
            if (first < last) {
                kt0 = it.lo / KT + first;
                kt1 = it.lo / KT + last;
                part = first == 0 && last == units ? -1 : 2 * cta + (first == 0);
                return true;
            }
        }
        return false;
    }

    // The CTA that ends the item of the last stay.
    __device__ __forceinline__ int last_cta() const { return cta + (at - 1) / per; }
};

// One row by one warp, key by key: for rows whose tile products met values that are
// not finite.  There a masked key's infinity or NaN times the zero of its weight
// would reach the row, so only keys that the row sees are touched here.  0.3 us a key, 0.85
// when all warps of an SM do rows of 200,000 keys; four keys at once were 1.4 times as fast, and
// their code made the others 2 % slower.
template <int D, int MODE>
__device__ __forceinline__ void paged_slow_row(const PagedArgs &a, const PagedItem &it, int row) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    __syncwarp();
    int lo, hi;
    paged_row_range(a, it, row, lo, hi);
    const int64_t qa = paged_row_offset(a, it, row, a.q_row, a.q_head) + lane * V;
    auto value = [](const uint16_t *p) {
        return MODE == PAGED_BF16 ? bf16_bits_to_f32(*p) : __half2float(*reinterpret_cast<const __half *>(p));
    };
    float q[V], o[V], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        q[i] = MODE == PAGED_F32 ? static_cast<const float *>(a.q)[qa + i] : value(static_cast<const uint16_t *>(a.q) + qa + i);
        o[i] = 0.0f;
    }
    for (int key = lo; key < hi; ++key) {
        const int page = a.table[it.b * a.table_ld + (key >> a.page_shift)];
        const bool ok = page >= 0 && page < a.pool;
        const int64_t s = key & ((1 << a.page_shift) - 1);
        const uint16_t *k = a.k + page * a.ks.page + s * a.ks.slot + it.h * a.ks.head + lane * V;
        const uint16_t *v = a.v + page * a.vs.page + s * a.vs.slot + it.h * a.vs.head + lane * V;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) x = fmaf(q[i], ok ? value(k + i) : 0.0f, x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        x *= a.scale_log2;
        const float top = x > m || x != x ? x : m;
        const float base = top == -INFINITY ? 0.0f : top;
        const float back = exp2_fast(m - base), p = exp2_fast(x - base);
        m = top;
        l = l * back + p;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = o[i] * back + p * (ok ? value(v + i) : 0.0f);
    }
    const int64_t at = paged_row_offset(a, it, row, a.out_row, D) + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float y = o[i] / l;
        if (MODE == PAGED_F32)
            static_cast<float *>(a.out)[at + i] = y;
        else if (MODE == PAGED_BF16)
            static_cast<__nv_bfloat16 *>(a.out)[at + i] = __float2bfloat16_rn(y);
        else
            static_cast<__half *>(a.out)[at + i] = __float2half_rn(y);
    }
    __syncwarp();
}

// Zeros for the rows of no request, by block column x: those before the first and behind the
// last.  Where a request does not fit, also the rows that it would have, and as its offsets may
// then lie anywhere, no row that some request which fits has (the block looks each row up).
template <int D, int MODE>
__device__ __forceinline__ void paged_zero_rows(const PagedArgs &a) {
    const int64_t bytes = a.out_row * (MODE == PAGED_F32 ? 4 : 2);
    auto any_request = [&](auto test) {
        bool hit = false;
        for (int b = threadIdx.x; b < a.requests; b += blockDim.x) hit |= test(paged_request(a, b));
        return __syncthreads_or(hit) != 0;
    };
    const bool bad = any_request([](const PagedRequest &r) { return r.bad; });
    const int64_t r0 = bad || !a.requests ? a.rows : a.starts[0], r1 = bad || !a.requests ? a.rows : a.starts[a.requests];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (row >= r0 && row < r1) {  // (the first row from r1 on that is this block's)
            row += (r1 - 1 - row) / gridDim.x * gridDim.x;
            continue;
        }
        if (bad && any_request([&](const PagedRequest &r) { return row >= r.row0 && row < r.row0 + int64_t{r.count}; })) continue;
        for (int64_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
            *reinterpret_cast<uint4 *>(static_cast<char *>(a.out) + row * bytes + i) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// ------------------------------------------------------------------ tiles
//
// Both attention kernels read K and V in tiles of 128 keys of one kv head, D / 64
// blocks of 128 rows of 64 values (128 bytes, 128-byte-swizzled), which the loading
// warps fetch by TMA, a lane to a box of one page piece and block, into a ring of
// stages that the other warps release.

constexpr int kTileKeys = 128;
// Rows of an item in the mma.sync kernel.  For fp16 and bf16 rows also the most that a
// request has there per kv head; more go to tcgen05 (32 fp16 requests over 4096 keys each,
// 128 columns: 16 rows take 99 us on mma.sync and 101 on tcgen05, 32 rows 115 and 102; 64
// requests over 2048 keys, 64 columns: 32 rows 81 and 100).
constexpr int kRowsItemMax = 64;
__host__ __device__ constexpr int rows_item(int head_dim, int mode) {
    return mode == PAGED_F32 ? kRowsItemMax : (head_dim == 64 ? 32 : 16);
}
constexpr int kTcItem = 256;  // tcgen05 kernel: two streams of 128
constexpr int kMaxStages = 8;
// Limit of a wait, more than a second.  Those in order are for the work on a tile or for the begin
// or end of a stay, microseconds at any length, or for rows that are done key by key, which
// may take long and are not counted (TileRing::slow).
constexpr uint32_t kTilePolls = 1u << 23;

template <int D>
constexpr int tile_bytes() {
    return kTileKeys * D * 2;
}

struct TileRing {
    uint64_t full[kMaxStages], empty[kMaxStages];
    volatile int abort;
    int slow;  // warps that do rows key by key
};

// Waits for phase `count` (0, 1, ..) of a barrier.  A wait that runs out sets `abort`,
// after which all waits pass: every role walks to its end.  Polls count only while no warp
// does rows key by key: that work ends by itself, but after a time that grows with the keys.
__device__ __forceinline__ bool tile_wait(TileRing &ring, uint64_t *b, uint32_t count) {
    for (uint32_t i = 0; i < kTilePolls; ++i) {
        if (mbar_try_wait(b, count & 1)) return true;
        if (ring.abort) return false;
        if (*const_cast<volatile int *>(&ring.slow)) i = 0;
    }
    ring.abort = 1;
    return false;
}
// tile_wait() by a whole warp, in branches that are the same for all lanes.
__device__ __forceinline__ bool warp_wait(TileRing &ring, uint64_t *b, uint32_t count) {
    for (uint32_t i = 0; i < kTilePolls; ++i) {
        if (__any_sync(0xffffffffu, mbar_try_wait(b, count & 1))) return true;
        if (__any_sync(0xffffffffu, ring.abort)) return false;
        if (__any_sync(0xffffffffu, *const_cast<volatile int *>(&ring.slow))) i = 0;
    }
    ring.abort = 1;
    return false;
}

// The rows of a stay (bit i: row0 + i) whose values are not finite, again, by the warp that did them.
template <int D, int MODE>
__device__ __forceinline__ void slow_rows(const PagedArgs &a, const PagedItem &it, TileRing &ring, int row0, unsigned odd) {
    if (!odd) return;
    const bool leader = (threadIdx.x & 31) == 0;
    if (leader) atomicAdd(&ring.slow, 1);
    for (; odd; odd &= odd - 1) paged_slow_row<D, MODE>(a, it, row0 + __ffs(odd) - 1);
    if (leader) atomicSub(&ring.slow, 1);
}
__device__ __forceinline__ void tile_arrive(uint64_t *b, uint32_t count = 1) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}

// The places in the ring of a stay's tiles, in order of use.  interleaved: keys and
// values of a tile one after the other; else the keys run two tiles ahead.
struct TileOrder {
    bool interleaved;
    int n;
    __device__ __forceinline__ int key_at(int j) const { return interleaved ? 2 * j : (j < 2 ? j : 2 * j - 1); }
    __device__ __forceinline__ int value_at(int j) const {
        if (interleaved) return 2 * j + 1;
        return n == 1 ? 1 : (j + 2 < n ? 2 * j + 2 : j + n);
    }
};

struct PagedMaps {
    CUtensorMap k, v;
    int heads_outer;  // coordinates (column, slot, head, page), else (column, head, slot, page)
};

// The whole run of loading warp `turn` of LOADERS, which have the tiles in turn: a warp
// issues the boxes of its lanes one after the other (about 130 cycles each), which at
// pages of 16 keys is longer than a tile takes to arrive.  A piece without a key that some
// row sees, or on a page outside the pool, is read as zeros (a box behind the last page).
template <int D, int STAGES, int LOADERS, typename Walk>
__device__ __forceinline__ void load_tiles(const PagedArgs &a, Walk &walk, TileRing &ring, uint8_t *stages,
                                           const CUtensorMap *k_map, const CUtensorMap *v_map, int heads_outer,
                                           int interleave_above, uint32_t turn) {
    const int lane = threadIdx.x & 31;
    asm volatile("fence.proxy.async.global;" ::: "memory");  // the cache rows that earlier kernels wrote
    const int piece = 1 << min(a.page_shift, 7);             // keys of a box
    const int pieces = kTileKeys / piece;
    const int block = lane / pieces, part = lane - block * pieces;
    uint32_t place = 0;
    // The copies of this warp in a range of places land before the CTA may end.
    auto land = [&](uint32_t from, uint32_t to, uint32_t polls) {
        for (uint32_t j = from; j < to; ++j)
            if (j % LOADERS == turn) mbar_wait_bounded(&ring.full[j % STAGES], (j / STAGES) & 1, polls);
    };
    PagedItem it;
    int kt0, kt1, out;
    while (walk.next(a, it, kt0, kt1, out)) {
        const TileOrder order{it.r1 - it.r0 > interleave_above, kt1 - kt0};
        const int32_t *table = a.table + it.b * a.table_ld;
        int next_key = 0, next_value = 0;
        for (int i = 0; i < 2 * order.n; ++i, ++place) {
            const bool value = next_key == order.n || order.value_at(next_value) == i;
            const int kt = kt0 + (value ? next_value++ : next_key++);
            if (place % LOADERS != turn) continue;
            const int key = kt * kTileKeys + part * piece;
            const bool seen = block < D / 64 && key < it.hi && key + piece > it.lo;
            int page = seen ? __ldg(table + (key >> a.page_shift)) : -1;
            const uint32_t s = place % STAGES;
            // After a wait ran out, stages are released before their tiles have come, so no further
            // copy may start; all lanes decide alike, since a stage's boxes are one transaction.
            if ((place >= STAGES && !warp_wait(ring, &ring.empty[s], place / STAGES - 1)) ||
                __any_sync(0xffffffffu, ring.abort)) {
                // this warp's copies may be one turn behind the ring's last STAGES places
                land(place > STAGES + LOADERS ? place - STAGES - LOADERS : 0, place, 1u << 16);
                return;
            }
            if (lane == 0) mbar_expect_tx(&ring.full[s], tile_bytes<D>());
            __syncwarp();
            if (block < D / 64) {
                if (page < 0 || page >= a.pool) {
                    if (seen) set_flag(a.flags, BD_FLAG_BAD_PAGE);
                    page = static_cast<int>(a.pool);
                }
                const int slot = key & ((1 << a.page_shift) - 1);
                asm volatile(
                    "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
                    "%5, %6}], [%2];" ::"r"(smem_u32(stages + s * tile_bytes<D>() + block * 16384 + part * piece * 128)),
                    "l"(value ? v_map : k_map), "r"(smem_u32(&ring.full[s])), "r"(block * 64),
                    "r"(heads_outer ? slot : it.h), "r"(heads_outer ? it.h : slot), "r"(page)
                    : "memory");
            }
            __syncwarp();
        }
    }
    // the last use of every stage (whoever reads these tiles waits for them too, but for a wait that ran out)
    land(place > STAGES ? place - STAGES : 0, place, kTilePolls);
}

// ------------------------------------------------------------------ launches

// Tensor maps of the caches; false when their strides cannot be expressed.
bool paged_maps(const PagedArgs &a, int head_dim, bool bf16, PagedMaps &maps);
int launch_paged_rows(const PagedArgs &a, const PagedMaps &maps, int head_dim, int mode, int ctas, cudaStream_t stream);
int launch_paged_tc(const PagedArgs &a, const PagedMaps &maps, int head_dim, int mode, int ctas, cudaStream_t stream);

}  // namespace bd
