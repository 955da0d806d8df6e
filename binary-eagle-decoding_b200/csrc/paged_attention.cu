// Attention of every request's new tokens over its keys in the paged cache:
//   o_t = sum_s p_ts v_s / sum_s p_ts,  p_ts = exp(scale q_t . k_s - m_t),
// over the keys s that token t (at position context + t) sees: s < context + count,
// s <= position when causal, |position - s| < window when windowed.  The seen keys of
// a token are one range [lo_t, hi_t).  Query heads in groups share a kv head: the
// rows of one (request, kv head) are its (token, head of the group) pairs, token
// major, so a kv head's keys are read once for all of them.
//
// One pass over the keys with a running maximum and sum per row; S = Q K^T and
// O = P V run on m16n8k16 MMAs with fp32 accumulators.  fp32 queries (over an fp16
// cache) enter as fp16 hi + lo halves of the row over a power of two, and P as hi +
// lo halves, which keeps about 22 bits of each.  fp16 and bf16 rows round P once to
// the cache's type (relative 2^-11 and 2^-8 at most, the size of the output's own
// rounding); the row sum adds the fp32 values.
//
// Work split: a unit is one 64-key tile of one item, an item is up to 64 rows of one
// (request, kv head).  The units of all items, in the order (request, head, rows,
// keys), are cut into equal ranges, one per resident CTA, so ragged batches and a
// single long request both load every SM alike.  An item that lies across CTAs
// leaves one partial (row maxima, sums, un-normalised O) per CTA in the workspace;
// a second launch joins them in CTA order.  Nothing waits on another CTA.
//
// The lengths are read on the device: no launch parameter depends on them.
#include "paged_attention.cuh"

namespace bd {

constexpr int kRowsThreads = 128;
constexpr int kRowsTile = 64;   // rows of an item
constexpr int kRowsKeys = 64;   // keys of a unit
constexpr int kRowsStages = 3;  // tiles in flight: 2 CTAs x 2 loading tiles x 32 KB cover the latency of HBM

template <int D>
constexpr size_t rows_smem() {
    return static_cast<size_t>(kRowsStages) * 2 * kRowsKeys * D * 2;
}

// 16-byte piece c of row r of a staged tile: pieces are permuted by the row so that
// the 8 rows of an ldmatrix lie in different banks.
template <int D>
__device__ __forceinline__ int piece(int r, int c) {
    return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

template <int MODE>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    if (MODE == PAGED_BF16)
        mma_bf16_16816(d, x[0], x[1], x[2], x[3], b0, b1);
    else
        mma_f16_16816(d, x[0], x[1], x[2], x[3], b0, b1);
}

template <int MODE>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if (MODE == PAGED_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// One CTA's stay on an item: key tiles [kt0, kt1) of it.  RW warps lie along the
// rows (16 each), 4 / RW along the keys of a tile, each with a maximum, sum and O of
// its own; they meet at the end through the staging area.
template <int D, int MODE, int RW>
__device__ __forceinline__ void rows_segment(const PagedArgs &a, const PagedItem &it, int kt0, int kt1, int part, char *sm) {
    constexpr int KW = 4 / RW, KK = kRowsKeys / KW;  // key parts, keys of a warp
    constexpr int kStage = 2 * kRowsKeys * D * 2;
    constexpr int kPieces = D / 8, kPass = kRowsThreads / kPieces;  // rows staged per pass of the CTA
    constexpr bool F32 = MODE == PAGED_F32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int rw = warp % RW, kw = warp / RW;

    // keys outside [lo, hi) are staged as zeros, whatever the cache holds there
    const int sc = tid % kPieces, sr = tid / kPieces;
    const int32_t *table = a.table + it.b * a.table_ld;
    auto stage = [&](int kt) {
        if (kt < kt1) {
            char *ks = sm + (kt % kRowsStages) * kStage, *vs = ks + kStage / 2;
            int page[kRowsKeys / kPass];
#pragma unroll
            for (int j = 0; j < kRowsKeys / kPass; ++j) {
                const int key = kt * kRowsKeys + sr + j * kPass;
                page[j] = key >= it.lo && key < it.hi ? __ldg(table + (key >> a.page_shift)) : -2;
            }
#pragma unroll
            for (int j = 0; j < kRowsKeys / kPass; ++j) {
                const int r = sr + j * kPass, key = kt * kRowsKeys + r;
                bool live = page[j] != -2;
                if (live && (page[j] < 0 || page[j] >= a.pool)) {
                    set_flag(a.flags, BD_FLAG_BAD_PAGE);
                    live = false;
                }
                const int64_t p = live ? page[j] : 0, s = key & ((1 << a.page_shift) - 1);
                cp_async16(ks + piece<D>(r, sc), a.k + p * a.ks.page + s * a.ks.slot + it.h * a.ks.head + sc * 8,
                           live ? 16 : 0);
                cp_async16(vs + piece<D>(r, sc), a.v + p * a.vs.page + s * a.vs.slot + it.h * a.vs.head + sc * 8,
                           live ? 16 : 0);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < kRowsStages - 1; ++s) stage(kt0 + s);

    // Q fragments of rows g and g + 8 of this warp, and the keys that they see
    uint32_t qh[D / 16][4], ql[F32 ? D / 16 : 1][4];
    float fold[2];  // scale x log2 e x the row's power of two
    int lo[2], hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = it.r0 + rw * 16 + g + 8 * r;
        const bool live = row < it.r1;
        paged_row_range(a, it, row, lo[r], hi[r]);
        const int64_t at = live ? paged_row_offset(a, it, row, a.q_row, a.q_head) : 0;
        fold[r] = a.scale_log2;
        if (F32) {
            const float *q = static_cast<const float *>(a.q) + at;
            float2 x[D / 16][2];
            float big = 0.0f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[s][j] = live ? *reinterpret_cast<const float2 *>(q + s * 16 + 8 * j + 2 * t) : make_float2(0.0f, 0.0f);
                    big = fmaxf(big, fmaxf(fabsf(x[s][j].x), fabsf(x[s][j].y)));
                }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // the halves of values up to 1 lose nothing to fp16's range
            int e = 0;
            if (big > 0.0f && big < INFINITY) e = min(max(ilogbf(big) + 1, -100), 126);
            const float down = ldexpf(1.0f, -e);
            fold[r] *= ldexpf(1.0f, e);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    split_half2(x[s][j].x * down, x[s][j].y * down, qh[s][r + 2 * j], ql[F32 ? s : 0][r + 2 * j]);
        } else {
            const uint16_t *q = static_cast<const uint16_t *>(a.q) + at;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    qh[s][r + 2 * j] = live ? *reinterpret_cast<const uint32_t *>(q + s * 16 + 8 * j + 2 * t) : 0u;
        }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

    for (int kt = kt0; kt < kt1; ++kt) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(kRowsStages - 2) : "memory");
        __syncthreads();  // tile kt has landed for all, and all are done with the stage that is loaded next
        stage(kt + kRowsStages - 1);
        const char *ks = sm + (kt % kRowsStages) * kStage, *vs = ks + kStage / 2;
        const int mi = lane >> 3, r8 = lane & 7;
        float s[KK / 8][4];
#pragma unroll
        for (int n = 0; n < KK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int n = 0; n < KK / 8; ++n) {
                uint32_t b[4];
                ldmatrix_x4(b, ks + piece<D>(kw * KK + n * 8 + r8, d * 4 + mi));
                mma16<MODE>(s[n], qh[2 * d], b[0], b[1]);
                mma16<MODE>(s[n], qh[2 * d + 1], b[2], b[3]);
                if (F32) {
                    mma16<MODE>(s[n], ql[F32 ? 2 * d : 0], b[0], b[1]);
                    mma16<MODE>(s[n], ql[F32 ? 2 * d + 1 : 0], b[2], b[3]);
                }
            }
        const int key0 = kt * kRowsKeys + kw * KK + 2 * t;
        const bool whole = kt * kRowsKeys >= it.lo_all && (kt + 1) * kRowsKeys <= it.hi_all;
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < KK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i >> 1, key = key0 + n * 8 + (i & 1);
                float x = s[n][i] * fold[r];
                if (!whole && (key < lo[r] || key >= hi[r])) x = -INFINITY;
                s[n][i] = x;
                top[r] = fmaxf(top[r], x);
            }
        float back[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            const float base = top[r] == -INFINITY ? 0.0f : top[r];  // no key seen yet: every term is 2^-inf = 0
            back[r] = exp2_fast(m[r] - base);
            m[r] = top[r];
            top[r] = base;
            l[r] *= back[r];
        }
#pragma unroll
        for (int n = 0; n < KK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = exp2_fast(s[n][i] - top[i >> 1]);
                l[i >> 1] += s[n][i];
            }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= back[i >> 1];
#pragma unroll
        for (int k = 0; k < KK / 16; ++k) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = s[2 * k + (j >> 1)][2 * (j & 1)], y = s[2 * k + (j >> 1)][2 * (j & 1) + 1];
                if (F32)
                    split_half2(x, y, ph[j], pl[j]);
                else
                    ph[j] = pack2<MODE>(x, y);
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, vs + piece<D>(kw * KK + k * 16 + (mi & 1) * 8 + r8, n * 2 + (mi >> 1)));
                mma16<MODE>(o[2 * n], ph, b[0], b[1]);
                mma16<MODE>(o[2 * n + 1], ph, b[2], b[3]);
                if (F32) {
                    mma16<MODE>(o[2 * n], pl, b[0], b[1]);
                    mma16<MODE>(o[2 * n + 1], pl, b[2], b[3]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();  // the staging area is free
    if (KW > 1) {
        // key parts 1.. hand their state to part 0, which adds them in order
        constexpr int kX = D / 8 * 4 + 4;
        float *x = reinterpret_cast<float *>(sm) + (rw * (KW - 1) * kX) * 32 + lane;
        if (kw > 0) {
            float *w = x + (kw - 1) * kX * 32;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[(n * 4 + i) * 32] = o[n][i];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                w[(kX - 4 + r) * 32] = m[r];
                w[(kX - 2 + r) * 32] = l[r];
            }
        }
        __syncthreads();
        if (kw == 0) {
#pragma unroll
            for (int p = 0; p < KW - 1; ++p) {
                const float *w = x + p * kX * 32;
                float mine[2], other[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float m1 = w[(kX - 4 + r) * 32], mx = fmaxf(m[r], m1), base = mx == -INFINITY ? 0.0f : mx;
                    mine[r] = exp2_fast(m[r] - base);
                    other[r] = exp2_fast(m1 - base);
                    l[r] = l[r] * mine[r] + w[(kX - 2 + r) * 32] * other[r];
                    m[r] = mx;
                }
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[n][i] = o[n][i] * mine[i >> 1] + w[(n * 4 + i) * 32] * other[i >> 1];
            }
        }
    }
    if (kw == 0) {
        bool odd[2] = {false, false};  // a value that is not finite
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = it.r0 + rw * 16 + g + 8 * r;
            if (row >= it.r1) continue;
            if (part >= 0) {
                const int64_t at = static_cast<int64_t>(part) * kRowsTile + row - it.r0;
                float *po = a.part_o + at * D;
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2 *>(po + n * 8 + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if (t == 0) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = make_float2(m[r], l[r]);
                continue;
            }
            const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
            const int64_t at = paged_row_offset(a, it, row, a.out_row, D);
            float probe = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                const float x = o[n][2 * r] * inv, y = o[n][2 * r + 1] * inv;
                probe += 0.0f * x + 0.0f * y;
                if (F32)
                    *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + n * 8 + 2 * t) = make_float2(x, y);
                else
                    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at + n * 8 + 2 * t) = pack2<MODE>(x, y);
            }
            odd[r] = !(probe == 0.0f);
        }
        // rows with a value that is not finite are done again, key by key
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            unsigned rows = __ballot_sync(0xffffffffu, odd[r]);
            while (rows) {
                const int gg = (__ffs(rows) - 1) >> 2;
                rows &= ~(0xFu << (4 * gg));
                paged_slow_row<D, MODE>(a, it, it.r0 + rw * 16 + gg + 8 * r);
            }
        }
    }
    __syncthreads();  // the exchange area is free for the next stay
}

template <int D, int MODE>
__global__ void __launch_bounds__(kRowsThreads, 2) paged_rows_kernel(const PagedArgs a) {
    extern __shared__ __align__(128) char paged_sm[];
    __shared__ PagedShared sh;
    grid_wait();
    grid_launch_dependents();
    PagedWalk<kRowsTile, kRowsKeys> walk;
    if (!walk.begin(a, sh, blockIdx.x, gridDim.x)) return;
    while (walk.more()) {
        PagedItem it;
        int kt0, kt1, part;
        walk.take(a, it, kt0, kt1, part);
        const int rows = it.r1 - it.r0;
        if (rows <= 16)
            rows_segment<D, MODE, 1>(a, it, kt0, kt1, part, paged_sm);
        else if (rows <= 32)
            rows_segment<D, MODE, 2>(a, it, kt0, kt1, part, paged_sm);
        else
            rows_segment<D, MODE, 4>(a, it, kt0, kt1, part, paged_sm);
    }
}

// Joins the partials of the items that lie across CTAs.  CTA (x, y) looks at the
// border between the ranges of CTAs x and x + 1 of the first launch: if it is the
// first one inside an item, it adds that item's partials in CTA order, a warp per row.
// y is the block of 8 rows.  It also zeroes the rows that belong to no request when
// the output is the library's caller's to define (zero_fill).
constexpr int kJoinThreads = 256;

template <int D, int MODE, int M, int KT>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a, int ctas) {
    __shared__ PagedShared sh;
    grid_wait();
    grid_launch_dependents();
    if (a.zero_fill && blockIdx.y == 0) paged_zero_rows<D, MODE>(a);
    PagedWalk<M, KT> walk;
    PagedItem it;
    int first, last;
    if (!walk.border(a, sh, blockIdx.x + 1, ctas, it, first, last)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = it.r0 + blockIdx.y * (kJoinThreads / 32) + warp;
    if (row >= it.r1) return;
    constexpr int V = D / 32;  // values of a lane
    auto place = [&](int p) { return (static_cast<int64_t>(2 * p + (p == first)) * M + row - it.r0); };
    float m = -INFINITY;
    for (int p = first + lane; p <= last; p += 32) m = fmaxf(m, a.part_ml[place(p) * 2]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
    for (int p0 = first; p0 <= last; p0 += 32) {
        float w = 0.0f, lw = 0.0f;
        if (p0 + lane <= last) {
            const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + place(p0 + lane) * 2);
            w = exp2_fast(ml.x - base);
            lw = w * ml.y;
        }
        const int n = min(32, last - p0 + 1);
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            l += __shfl_sync(0xffffffffu, lw, j);
            const float *po = a.part_o + place(p0 + j) * D + lane * V;
            if (V == 4) {
                const float4 x = *reinterpret_cast<const float4 *>(po);
                o[0] += wj * x.x;
                o[1] += wj * x.y;
                o[V - 2] += wj * x.z;
                o[V - 1] += wj * x.w;
            } else {
                const float2 x = *reinterpret_cast<const float2 *>(po);
                o[0] += wj * x.x;
                o[1] += wj * x.y;
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = paged_row_offset(a, it, row, a.out_row, D) + lane * V;
    float probe = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        o[i] *= inv;
        probe += 0.0f * o[i];
    }
    if (__any_sync(0xffffffffu, !(probe == 0.0f))) {
        paged_slow_row<D, MODE>(a, it, row);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        if (MODE == PAGED_F32)
            *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + i) = make_float2(o[i], o[i + 1]);
        else if (MODE == PAGED_BF16)
            *reinterpret_cast<__nv_bfloat162 *>(static_cast<uint16_t *>(a.out) + at + i) = __floats2bfloat162_rn(o[i], o[i + 1]);
        else
            *reinterpret_cast<__half2 *>(static_cast<uint16_t *>(a.out) + at + i) = __floats2half2_rn(o[i], o[i + 1]);
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

template <int D, int MODE>
static int launch_rows(const PagedArgs &a, cudaStream_t stream) {
    const int ctas = 2 * device_sms();
    if (cudaFuncSetAttribute(paged_rows_kernel<D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(rows_smem<D>())) != cudaSuccess)
        return BD_ERR_LAUNCH;
    const int st = launch_pdl(paged_rows_kernel<D, MODE>, dim3(ctas), dim3(kRowsThreads), rows_smem<D>(), stream, a);
    if (st) return st;
    return launch_pdl(paged_join_kernel<D, MODE, kRowsTile, kRowsKeys>, dim3(ctas - 1, kRowsTile / (kJoinThreads / 32)),
                      dim3(kJoinThreads), 0, stream, a, ctas);
}

}  // namespace bd

using namespace bd;

static size_t rows_partials(int ctas) { return static_cast<size_t>(2) * ctas * kRowsTile; }

extern "C" size_t bd_paged_attention_workspace_bytes(int head_dim) {
    return rows_partials(2 * device_sms()) * (head_dim + 2) * sizeof(float) + 256;
}

extern "C" int bd_paged_attention(const bd_paged_attention_args *p, bd_stream_t stream) {
    if (!p || p->requests < 0 || p->rows < 0 || p->rows > INT32_MAX || p->kv_heads < 1 || p->heads < 1 ||
        p->heads % p->kv_heads || p->heads > 65535 || (p->head_dim != 64 && p->head_dim != 128) ||
        !page_size_ok(p->page_size) || !pool_ok(p->pool_pages, p->page_size) ||
        !table_ok(p->table_width, p->page_size) || p->table_ld < p->table_width || p->window < 0 ||
        p->longest < 0 || !(p->scale > -INFINITY && p->scale < INFINITY))
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
    if (!p->workspace || p->workspace_bytes < bd_paged_attention_workspace_bytes(p->head_dim)) return BD_ERR_WORKSPACE;
    PagedArgs a{};
    if (!cache_strides(p->k_strides, a.ks) || !cache_strides(p->v_strides, a.vs)) return BD_ERR_ALIGNMENT;
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
    a.groups = p->heads / p->kv_heads;
    a.page_shift = log2_of(p->page_size);
    a.causal = p->causal != 0;
    a.window = p->window > INT32_MAX ? 0 : static_cast<int>(p->window);
    a.longest = p->longest ? p->longest : INT32_MAX;
    a.scale_log2 = p->scale * 1.4426950408889634f;  // log2 e
    a.out = p->out;
    a.out_row = static_cast<int64_t>(p->heads) * p->head_dim;
    a.zero_fill = p->zero_fill;
    a.part_o = static_cast<float *>(p->workspace);
    a.part_ml = a.part_o + rows_partials(2 * device_sms()) * p->head_dim;
    a.flags = p->flags;
    if (p->head_dim == 64)
        return mode == PAGED_F32   ? launch_rows<64, PAGED_F32>(a, stream)
               : mode == PAGED_F16 ? launch_rows<64, PAGED_F16>(a, stream)
                                   : launch_rows<64, PAGED_BF16>(a, stream);
    return mode == PAGED_F32   ? launch_rows<128, PAGED_F32>(a, stream)
           : mode == PAGED_F16 ? launch_rows<128, PAGED_F16>(a, stream)
                               : launch_rows<128, PAGED_BF16>(a, stream);
}
