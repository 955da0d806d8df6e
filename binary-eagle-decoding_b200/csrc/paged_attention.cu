// Attention of every request's new tokens over its keys in the paged cache:
//   o_t = sum_s p_ts v_s / sum_s p_ts,  p_ts = exp(scale q_t . k_s - m_t),
// over the keys s that token t (at position context + t) sees: s < context + count,
// s <= position when causal, |position - s| < window when windowed.  The seen keys of
// a token are one range [lo_t, hi_t).  Query heads in groups share a kv head: the
// rows of one (request, kv head) are its (token, head of the group) pairs, token
// major, so a kv head's keys are read once for all of them.
//
// One pass over the keys with a running maximum and sum per row, S = Q K^T and
// O = P V on the tensor cores with fp32 accumulators.  fp32 queries (over an fp16
// cache) enter as fp16 hi + lo halves of the row times a power of two, and P as hi +
// lo halves.  fp16 and bf16 rows round P once to the cache's type (relative 2^-11 and 2^-8 at
// most, the size of the output's own rounding); the row sum adds the fp32 values.  fp16 has
// no step under 2^-24, so P is scaled up to 2^15 there: halves keep 22 bits of weights down to
// 2^-18 of the row's largest and an error of 2^-40 of it below; a rounded P its 2^-11 down to
// 2^-29 (tcgen05: 2^-25) and an error of 2^-40 (2^-36) below.
//
// Two kernels: requests of up to 16 rows per kv head (32 with 64 columns), and fp32 rows of
// any count, run on mma.sync (paged_attention_rows.cu), the others on tcgen05
// (paged_attention_tc.cu).  A batch may hold both kinds; lengths are read on the device,
// so no launch parameter depends on them.
//
// Work split, in each: a unit is one 128-key tile of one item, an item is up to M
// rows of one (request, kv head).  The units of all items, in the order (request,
// head, rows, keys), are cut into equal ranges, one per CTA and SM, so ragged batches
// and a single long request both load every SM alike.  An item that lies across CTAs
// leaves one partial (row maxima, sums, un-normalised O) per CTA in the workspace;
// a last launch joins them in CTA order.  Nothing waits on another CTA.
#include "paged_attention.cuh"

#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>

namespace bd {

// A batch that may hold longer requests pays 4 to 8 us for the mma.sync kernel's launch
// even if it has no rows there.  With up to 256 pairs all go to tcgen05 (two chunks of 1024
// tokens and 6 single tokens over 4096 keys, 8 kv heads: 149 us instead of 181, 14: 181 and
// 202, 30: 251 and 246, 62: 386 and 326; 32 x 17 tokens over 2048 keys: 76 and 84).
constexpr int kOneKernelPairs = 256;
constexpr float kLog2e = 1.4426950408889634f;

// Joins the partials of the items that lie across CTAs: CTA (x, y) those of the item
// that CTA x (of the first kernel, then of the second) left open, a warp to a row, 8
// rows of every 8 Y.  It also zeroes the rows that belong to no request when the
// output is the library's to define (zero_fill).
constexpr int kJoinThreads = 256;
constexpr int kJoinBlocks = 8;  // Y

template <int D, int MODE>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a, int ctas) {
    grid_wait();
    grid_launch_dependents();
    const int set = a.split_rows == 0 || blockIdx.x >= ctas, cta = blockIdx.x % ctas;
    const PagedArgs::Parts &parts = a.parts[set];
    const PagedOpen open = parts.open[cta];
    if (a.zero_fill && blockIdx.y == 0) paged_zero_rows<D, MODE>(a);
    if (open.last < 0) return;
    const PagedItem &it = open.it;
    const int rows = set ? kTcItem : a.item_rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int V = D / 32;  // values of a lane
    for (int row = it.r0 + blockIdx.y * (kJoinThreads / 32) + warp; row < it.r1; row += kJoinBlocks * (kJoinThreads / 32)) {
        auto place = [&](int p) { return static_cast<int64_t>(2 * p + (p == cta)) * rows + row - it.r0; };
        auto stats = [&](int p) {
            return p <= open.last ? *reinterpret_cast<const float2 *>(parts.ml + place(p) * 2) : make_float2(-INFINITY, 0.0f);
        };
        float2 ml = stats(cta + lane);
        float m = ml.x;
        for (int p = cta + 32 + lane; p <= open.last; p += 32) m = fmaxf(m, stats(p).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.0f;
        for (int p0 = cta; p0 <= open.last; p0 += 32) {
            if (p0 != cta) ml = stats(p0 + lane);
            const float w = exp2_fast(ml.x - base), lw = w * ml.y;
            const int n = min(32, open.last - p0 + 1);
            // O of eight partials in flight
            for (int j0 = 0; j0 < n; j0 += 8) {
                float x[8][V];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j0 + j >= n) break;
                    const float *po = parts.o + place(p0 + j0 + j) * D + lane * V;
                    if (V == 4)
                        *reinterpret_cast<float4 *>(x[j]) = *reinterpret_cast<const float4 *>(po);
                    else
                        *reinterpret_cast<float2 *>(x[j]) = *reinterpret_cast<const float2 *>(po);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j0 + j >= n) break;
                    const float wj = __shfl_sync(0xffffffffu, w, j0 + j);
                    l += __shfl_sync(0xffffffffu, lw, j0 + j);
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] += wj * x[j][i];
                }
            }
        }
        const float inv = 1.0f / l;  // l is 0 only when every seen score is -inf: not a number
        const int64_t at = paged_row_offset(a, it, row, a.out_row, D) + lane * V;
        float probe = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            o[i] *= inv;
            probe += 0.0f * o[i];
        }
        if (__any_sync(0xffffffffu, !(probe == 0.0f))) {
            paged_slow_row<D, MODE>(a, it, row);
            continue;
        }
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            if (MODE == PAGED_F32)
                *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + i) = make_float2(o[i], o[i + 1]);
            else if (MODE == PAGED_BF16)
                *reinterpret_cast<__nv_bfloat162 *>(static_cast<uint16_t *>(a.out) + at + i) = __floats2bfloat162_rn(o[i], o[i + 1]);
            else
                *reinterpret_cast<__half2 *>(static_cast<uint16_t *>(a.out) + at + i) =
                    __floats2half2_rn(paged_bounded<MODE>(o[i]), paged_bounded<MODE>(o[i + 1]));
        }
    }
}

static int device_sms() {
    static int cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!cached[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// A cache as (column, head, slot, page), or (column, slot, head, page) when heads lie
// further apart than slots; boxes of 64 columns and one page piece of one head.
static bool cache_map(CUtensorMap *m, const uint16_t *base, const CacheStrides &s, const PagedArgs &a, int head_dim, bool bf16,
                      bool heads_outer) {
    auto encode = map_encoder();
    if (!encode) return false;
    const cuuint32_t page = 1u << a.page_shift, box_rows = page < kTileKeys ? page : kTileKeys;
    const cuuint64_t heads = static_cast<cuuint64_t>(a.kv_heads);
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), heads_outer ? page : heads, heads_outer ? heads : page,
                                static_cast<cuuint64_t>(a.pool)};
    const int64_t inner = heads_outer ? s.slot : s.head, outer = heads_outer ? s.head : s.slot;
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(inner) * 2, static_cast<cuuint64_t>(outer) * 2,
                                   static_cast<cuuint64_t>(s.page) * 2};
    const cuuint32_t box[4] = {64, heads_outer ? box_rows : 1, heads_outer ? 1 : box_rows, 1};
    const cuuint32_t each[4] = {1, 1, 1, 1};
    return encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  const_cast<uint16_t *>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B,
                  // a row and no more: with 64 columns 256 bytes are two heads' rows, which other CTAs read
                  // at other times (131072 keys: 70 us, with 128 bytes 60)
                  head_dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool paged_maps(const PagedArgs &a, int head_dim, bool bf16, PagedMaps &maps) {
    maps.heads_outer = a.ks.head > a.ks.slot;  // one order of coordinates for both caches
    return cache_map(&maps.k, a.k, a.ks, a, head_dim, bf16, maps.heads_outer) &&
           cache_map(&maps.v, a.v, a.vs, a, head_dim, bf16, maps.heads_outer);
}

template <int D>
static int launch_join(const PagedArgs &a, int mode, int sets, int ctas, cudaStream_t stream) {
    const dim3 grid(sets * ctas, kJoinBlocks), block(kJoinThreads);
    if (mode == PAGED_F32) return launch_pdl(paged_join_kernel<D, PAGED_F32>, grid, block, 0, stream, a, ctas);
    if (mode == PAGED_F16) return launch_pdl(paged_join_kernel<D, PAGED_F16>, grid, block, 0, stream, a, ctas);
    return launch_pdl(paged_join_kernel<D, PAGED_BF16>, grid, block, 0, stream, a, ctas);
}

// The workspace: of each kernel the partials' O, maxima and sums, and the open items.
static size_t carve(PagedArgs &a, void *workspace, int head_dim) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *p = static_cast<char *>(workspace) + off;
        off += (bytes + 255) & ~static_cast<size_t>(255);
        return static_cast<void *>(p);
    };
    const size_t ctas = device_sms();
    for (int set = 0; set < 2; ++set) {
        const size_t rows = 2 * ctas * (set ? kTcItem : kRowsItemMax);
        a.parts[set].o = static_cast<float *>(take(rows * head_dim * sizeof(float)));
        a.parts[set].ml = static_cast<float *>(take(rows * 2 * sizeof(float)));
        a.parts[set].open = static_cast<PagedOpen *>(take(ctas * sizeof(PagedOpen)));
    }
    return off;
}

}  // namespace bd

using namespace bd;

extern "C" size_t bd_paged_attention_workspace_bytes(int head_dim) {
    PagedArgs a{};
    return carve(a, nullptr, head_dim);
}

extern "C" int bd_paged_attention(const bd_paged_attention_args *p, bd_stream_t stream) {
    if (!p || p->requests < 0 || p->rows < 0 || p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads ||
        p->heads > 65535 || p->rows > INT32_MAX / (p->heads / p->kv_heads) ||
        (p->head_dim != 64 && p->head_dim != 128) || !page_size_ok(p->page_size) ||
        !pool_ok(p->pool_pages, p->page_size) || !table_ok(p->table_width, p->page_size) ||
        p->table_ld < p->table_width || p->window < 0 || p->longest < 0 || !std::isfinite(p->scale * kLog2e))
        return BD_ERR_INVALID;
    int mode;
    if (p->row_type == BD_F32 && p->cache_type == BD_F16)
        mode = PAGED_F32;
    else if (p->row_type == BD_F16 && p->cache_type == BD_F16)
        mode = PAGED_F16;
    else if (p->row_type == BD_BF16 && p->cache_type == BD_BF16)
        mode = PAGED_BF16;
    else
        return BD_ERR_INVALID;
    if (p->rows == 0) return BD_OK;
    if (!p->q || !p->out || !p->k_cache || !p->v_cache || (p->requests && (!p->table || !p->context || !p->starts)))
        return BD_ERR_INVALID;
    const int64_t unit = mode == PAGED_F32 ? 4 : 8;
    if (!aligned16(p->q) || !aligned16(p->out) || !aligned16(p->k_cache) || !aligned16(p->v_cache) ||
        ((p->q_row | p->q_head) % unit) != 0)
        return BD_ERR_ALIGNMENT;
    PagedArgs a{};
    if (!cache_strides(p->k_strides, a.ks) || !cache_strides(p->v_strides, a.vs)) return BD_ERR_ALIGNMENT;
    if (!p->workspace || !aligned16(p->workspace) || p->workspace_bytes < carve(a, p->workspace, p->head_dim))
        return BD_ERR_WORKSPACE;
    a.q = p->q;
    a.q_row = p->q_row;
    a.q_head = p->q_head;
    a.k = static_cast<const uint16_t *>(p->k_cache);
    a.v = static_cast<const uint16_t *>(p->v_cache);
    a.table = p->table;
    a.table_ld = p->table_ld;
    a.table_width = p->table_width;
    a.pool = p->pool_pages;
    a.context = p->context;
    a.starts = p->starts;
    a.requests = p->requests;
    a.rows = p->rows;
    a.kv_heads = p->kv_heads;
    paged_set_groups(a, p->heads / p->kv_heads);
    a.page_shift = log2_of(p->page_size);
    a.causal = p->causal != 0;
    a.window = p->window > INT32_MAX ? 0 : static_cast<int>(p->window);
    a.longest = p->longest ? p->longest : INT32_MAX;
    a.scale_log2 = p->scale * kLog2e;
    a.out = p->out;
    a.out_row = static_cast<int64_t>(p->heads) * p->head_dim;
    a.zero_fill = p->zero_fill;
    a.flags = p->flags;
    // rows may be read after others are written
    const int64_t each = mode == PAGED_F32 ? 4 : 2, q_rows = (p->rows - 1) * p->q_row, q_heads = (p->heads - 1) * p->q_head;
    const int64_t q_first = std::min<int64_t>(q_rows, 0) + std::min<int64_t>(q_heads, 0);
    const Span out = span_of(p->out, p->rows * a.out_row * each);
    if (out.meets(span_of(static_cast<const char *>(p->q) + q_first * each,
                          (std::max<int64_t>(q_rows, 0) + std::max<int64_t>(q_heads, 0) - q_first + p->head_dim) * each)) ||
        out.meets(cache_span(p->k_cache, a.ks, a.pool, p->page_size, a.kv_heads, p->head_dim)) ||
        out.meets(cache_span(p->v_cache, a.vs, a.pool, p->page_size, a.kv_heads, p->head_dim)) ||
        (a.requests && (out.meets(span_of(p->table, 4 * ((a.requests - 1) * p->table_ld + p->table_width))) ||
                        out.meets(span_of(p->context, 4 * int64_t{a.requests})) ||
                        out.meets(span_of(p->starts, 4 * (int64_t{a.requests} + 1))))) ||
        out.meets(span_of(p->workspace, static_cast<int64_t>(p->workspace_bytes))))
        return BD_ERR_INVALID;
    const int64_t pairs = static_cast<int64_t>(a.requests) * a.kv_heads;
    a.item_rows = rows_item(p->head_dim, mode);
    a.split_rows = mode == PAGED_F32 ? INT_MAX : a.item_rows;
    // a batch that cannot hold a longer request needs the one kernel
    const bool tiles = std::min<int64_t>(a.longest, p->rows) * a.groups > a.split_rows;
    const bool few = !tiles || pairs > kOneKernelPairs;
    if (!few) a.split_rows = 0;  // the tcgen05 kernel has them all
    PagedMaps maps;
    if (!paged_maps(a, p->head_dim, mode == PAGED_BF16, maps)) return BD_ERR_ALIGNMENT;
    const int ctas = device_sms();
    int st = few ? launch_paged_rows(a, maps, p->head_dim, mode, ctas, stream) : BD_OK;
    if (!st && tiles) st = launch_paged_tc(a, maps, p->head_dim, mode, ctas, stream);
    if (st) return st;
    return p->head_dim == 64 ? launch_join<64>(a, mode, few + tiles, ctas, stream)
                             : launch_join<128>(a, mode, few + tiles, ctas, stream);
}
