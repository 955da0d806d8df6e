// Work split and row helpers of the paged attention, shared by its kernels.
#pragma once

#include "paged.cuh"

namespace bd {

enum PagedMode : int {
    PAGED_F32 = 0,   // fp32 rows over an fp16 cache
    PAGED_F16 = 1,   // fp16 rows and cache
    PAGED_BF16 = 2,  // bf16 rows and cache
};

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
    int causal, window, longest;  // window 0: none
    float scale_log2;             // scale x log2 e
    void *out;
    int64_t out_row;  // heads stand head_dim apart
    int zero_fill;
    float *part_o, *part_ml;  // [2 x CTAs][rows of an item][head_dim], [..][2]
    int32_t *flags;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
    paged_token_range(a, r.context, r.count, it.r0 / a.groups, it.lo, it.hi_all);
    paged_token_range(a, r.context, r.count, (it.r1 - 1) / a.groups, it.lo_all, it.hi);
}

__device__ __forceinline__ void paged_row_range(const PagedArgs &a, const PagedItem &it, int row, int &lo, int &hi) {
    if (row < it.r1) {
        paged_token_range(a, it.context, it.count, row / a.groups, lo, hi);
    } else {
        lo = hi = 0;
    }
}

// Element offset of a row in a tensor of the given token and head strides.
__device__ __forceinline__ int64_t paged_row_offset(const PagedArgs &a, const PagedItem &it, int row, int64_t token_stride,
                                                    int64_t head_stride) {
    const int t = row / a.groups;
    return (static_cast<int64_t>(it.row0) + t) * token_stride +
           (static_cast<int64_t>(it.h) * a.groups + (row - t * a.groups)) * head_stride;
}

struct PagedShared {
    int64_t warp_sums[32];
    int64_t before;
    int b;
};

// The walk over the units of this CTA's range, see the head of paged_attention.cu.
// M rows to an item, KT keys to a unit.  Requests of more than `above` rows (0: all)
// are walked, or of at most `upto` rows.
template <int M, int KT>
struct PagedWalk {
    int64_t u, end, total, per;
    int cta, off;          // off: units of the current item before u
    int b, h, i, tiles, units;  // units: of the item
    PagedRequest r;
    PagedItem it;

    static __device__ __forceinline__ int item_units(const PagedItem &x) { return (x.hi + KT - 1) / KT - x.lo / KT; }

    // Units of one kv head of request b.
    static __device__ __forceinline__ int64_t request_units(const PagedArgs &a, int b) {
        const PagedRequest r = paged_request(a, b);
        if (r.bad) set_flag(a.flags, BD_FLAG_BAD_LENGTH);
        const int tiles = (r.count * a.groups + M - 1) / M;
        int64_t sum = 0;
        for (int i = 0; i < tiles; ++i) {
            PagedItem x;
            paged_item<M>(a, r, i, x);
            sum += item_units(x);
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
        tiles = (r.count * a.groups + M - 1) / M;
    }
    __device__ __forceinline__ void set_item(const PagedArgs &a) {
        paged_item<M>(a, r, i, it);
        it.b = b;
        it.h = h;
        units = item_units(it);
    }

    // Places the walk at unit `cta x per` of `ctas` equal ranges; false when the range is empty.
    __device__ __forceinline__ bool begin(const PagedArgs &a, PagedShared &sh, int cta_, int ctas) {
        cta = cta_;
        const int n = blockDim.x, tid = threadIdx.x;
        int64_t w = tid < a.requests ? request_units(a, tid) * a.kv_heads : 0, sum;
        int64_t incl = scan(w, sh, sum);
        total = sum;
        for (int b0 = n; b0 < a.requests; b0 += n) {
            scan(b0 + tid < a.requests ? request_units(a, b0 + tid) * a.kv_heads : 0, sh, sum);
            total += sum;
        }
        per = (total + ctas - 1) / ctas;
        u = cta * per;
        end = min(u + per, total);
        if (u >= end) return false;
        // the request that holds unit u
        int64_t before = 0;
        for (int b0 = 0; b0 < a.requests; b0 += n) {
            if (b0 > 0 || a.requests > n) {
                w = b0 + tid < a.requests ? request_units(a, b0 + tid) * a.kv_heads : 0;
                incl = scan(w, sh, sum);
            }
            if (before + incl - w <= u && u < before + incl) {
                sh.b = b0 + tid;
                sh.before = before + incl - w;
            }
            before += sum;
            if (u < before) break;
        }
        __syncthreads();
        b = sh.b;
        int64_t rest = u - sh.before;
        set_request(a);
        // its kv head and rows
        int64_t each = 0;
        for (int j = 0; j < tiles; ++j) {
            paged_item<M>(a, r, j, it);
            each += item_units(it);
        }
        h = static_cast<int>(rest / each);
        rest -= h * each;
        for (i = 0;; ++i) {
            set_item(a);
            if (rest < units) break;
            rest -= units;
        }
        off = static_cast<int>(rest);
        return true;
    }

    __device__ __forceinline__ bool more() const { return u < end; }

    // The next stay: an item, its key tiles [kt0, kt1), and the partial it leaves (-1: it is done whole).
    __device__ __forceinline__ void take(const PagedArgs &a, PagedItem &item, int &kt0, int &kt1, int &part) {
        item = it;
        const int n = static_cast<int>(min(static_cast<int64_t>(units - off), end - u));
        kt0 = it.lo / KT + off;
        kt1 = kt0 + n;
        part = off == 0 && n == units ? -1 : 2 * cta + (off == 0);
        u += n;
        if (u >= end) return;
        off = 0;
        if (++i == tiles) {
            i = 0;
            if (++h == a.kv_heads) {
                h = 0;
                do {
                    ++b;
                    set_request(a);
                } while (tiles == 0);
            }
        }
        set_item(a);
    }

    // The item around the border before range c, if that border is the first one inside it;
    // its partials are those of CTAs first .. last.
    __device__ __forceinline__ bool border(const PagedArgs &a, PagedShared &sh, int c, int ctas, PagedItem &item, int &first,
                                           int &last) {
        if (!begin(a, sh, c, ctas) || off == 0) return false;
        const int64_t start = u - off;
        if ((c - 1) * per > start) return false;
        item = it;
        first = c - 1;
        last = static_cast<int>((start + units - 1) / per);
        return true;
    }
};

// One row by one warp, key by key: for rows whose tile products met values that are
// not finite.  There a masked key's infinity or NaN times the zero of its weight
// would reach the row, so only keys that the row sees are touched here.
template <int D, int MODE>
__device__ __noinline__ void paged_slow_row(const PagedArgs &a, const PagedItem &it, int row) {
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
        const float y = l == 0.0f ? 0.0f : o[i] / l;
        if (MODE == PAGED_F32)
            static_cast<float *>(a.out)[at + i] = y;
        else if (MODE == PAGED_BF16)
            static_cast<__nv_bfloat16 *>(a.out)[at + i] = __float2bfloat16_rn(y);
        else
            static_cast<__half *>(a.out)[at + i] = __float2half_rn(y);
    }
    __syncwarp();
}

// Zeros for the rows of no request: before the first, behind the last, of a refused one.
template <int D, int MODE>
__device__ __forceinline__ void paged_zero_rows(const PagedArgs &a) {
    const int64_t bytes = a.out_row * (MODE == PAGED_F32 ? 4 : 2);
    auto zero = [&](int64_t r0, int64_t r1, int64_t step) {
        for (int64_t r = r0; r < r1; r += step)
            for (int64_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
                *reinterpret_cast<uint4 *>(static_cast<char *>(a.out) + r * bytes + i) = make_uint4(0u, 0u, 0u, 0u);
    };
    auto clamp = [&](int64_t r) { return r < 0 ? int64_t{0} : (r > a.rows ? a.rows : r); };
    const int64_t r0 = a.requests ? clamp(a.starts[0]) : 0, r1 = a.requests ? clamp(a.starts[a.requests]) : 0;
    zero(blockIdx.x, r0, gridDim.x);
    zero(r1 + blockIdx.x, a.rows, gridDim.x);
    for (int b = blockIdx.x; b < a.requests; b += gridDim.x)
        if (paged_request(a, b).bad) zero(clamp(a.starts[b]), clamp(a.starts[b + 1]), 1);
}

}  // namespace bd
