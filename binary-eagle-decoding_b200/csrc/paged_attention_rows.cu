// Attention over the paged cache for few rows per (request, kv head), as of single
// tokens, and for fp32 rows of any count.  The mathematics and the work split are
// those at the head of paged_attention.cu, with 16, 32 or 64 rows to an item.
//
// One CTA per SM: four warps load key and value tiles by TMA into a ring of six
// stages (about 190 KB in flight, which is what covers HBM's latency), eight warps
// compute.  RW of them lie along the rows (16 each), 8 / RW along the keys of a
// tile; each has the running maximum, sum and O of its rows over its keys, so the
// warps meet only at the end of a stay.  S = Q K^T and O += P V are m16n8k16 MMAs.
// At one token and four heads to a kv head the MMAs, softmax and loads of a warp
// hide under the 2800 cycles that a tile takes to come from HBM: 64 requests over 1024 to
// 8192 keys (1.09 GB) take 171 us = 6.4 TB/s, one over 131072 keys 94 us = 5.7 TB/s.
// fp32 rows do twice the MMAs and are bound by these and by the chain through a tile from
// 64 rows on: 24 draft blocks in a window of 4096 take 169 us, 54 % of the MMA pipe.
#include "paged_attention.cuh"

namespace bd {

constexpr int kRowsWarps = 8;
constexpr int kPlane = 64;  // rows of a plane of Q in shared memory
// A stay's Q, joining and output, in units.  Other batches than those above: 64 tokens over 291,000
// keys (1.19 GB) take 199 us with 1, 189 with 2, 184 with 4, of 64 columns 123, 118 and 113; 24
// draft blocks over 1024 to 8192 keys in a window of 4096 take 170, 163 and 162, over 4096
// keys each 184, 180 and 180, where 2 and 4 do not differ.
template <int D, int MODE>
constexpr int rows_extra() {
    return MODE == PAGED_F32 && D == 128 ? 2 : 4;
}
constexpr int kRowsThreads = 384;

template <int D>
constexpr int rows_stages() {
    return D == 128 ? 6 : 8;
}
// Q of an item (fp32 rows: two planes), and at the end of a stay what half the warps
// hand to the other half: of 4 warps, O (32 lanes x D / 2 floats) and (m, l) of 16 rows.
template <int D>
constexpr int rows_area() {
    return 4 * (32 * (D / 2) + 16 * 2) * 4;
}
template <int D>
constexpr size_t rows_smem() {
    return 1024 + static_cast<size_t>(rows_stages<D>()) * tile_bytes<D>() + rows_area<D>();
}
static_assert(rows_smem<128>() + sizeof(TileRing) + 1024 <= 232448, "one CTA's shared memory");
static_assert(rows_area<128>() >= 2 * kPlane * 128 * 2 && rows_area<64>() >= 2 * kPlane * 64 * 2, "Q fits");

struct RowsShared {
    TileRing ring;
    float fold[kPlane];
    PagedShared walk;
};

// 16-byte piece c of row r of a staged tile or plane of R rows (128-byte-swizzled blocks of 64 columns).
template <int R>
__device__ __forceinline__ uint32_t tile_piece(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * (R * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
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

// The weights of fp16 caches enter the products times 2^15 (at most 32768), which leaves fp16's whole
// range below them: unscaled, every weight under 2^-25 of the largest was lost to O and not to
// the sum (8192 keys 18 nats below one of small value: up to a third of the output).
template <int MODE>
constexpr float rows_weight_scale() {
    return MODE == PAGED_BF16 ? 1.0f : 32768.0f;
}

__device__ __forceinline__ void rows_meet() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The Q rows of an item into shared memory, four threads to a row.  fp32 rows are scaled by a
// power of two that takes the row's largest value to 2^14 .. 2^15, fp16's upper end, so that
// the halves hold values down to 2^-17 of the largest with 22 bits and smaller ones within
// 2^-39 of it (scaled to 1, a row's values under 2^-25 of its largest were 0); fold = scale x
// log2 e over that power.
template <int D, int MODE>
__device__ __forceinline__ void rows_load_q(const PagedArgs &a, const PagedItem &it, uint8_t *area, RowsShared &sh) {
    constexpr int kChunks = D / 32;  // 16-byte pieces (of 16-bit values) of a thread
    const int r = threadIdx.x >> 2, part = threadIdx.x & 3, row = it.r0 + r;
    const bool live = row < it.r1;
    if (it.r0 + (r & ~15) >= it.r1) return;  // no live row in its 16 (two whole warps): never read
    const int64_t at = (live ? paged_row_offset(a, it, row, a.q_row, a.q_head) : 0) + part * kChunks * 8;
    if (MODE == PAGED_F32) {
        const float *q = static_cast<const float *>(a.q) + at;
        float4 x[kChunks * 2];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < kChunks * 2; ++i) {
            x[i] = live ? __ldg(reinterpret_cast<const float4 *>(q) + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            big = fmaxf(big, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        int e = 0;
        if (big > 0.0f && big < INFINITY) e = max(ilogbf(big) + 1, -100) - 15;
        const float down = ldexpf(1.0f, -e);
        if (part == 0) sh.fold[r] = a.scale_log2 * ldexpf(1.0f, e);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const float4 u = x[2 * i], v = x[2 * i + 1];
            uint4 hi, lo;
            split_half2(u.x * down, u.y * down, hi.x, lo.x);
            split_half2(u.z * down, u.w * down, hi.y, lo.y);
            split_half2(v.x * down, v.y * down, hi.z, lo.z);
            split_half2(v.z * down, v.w * down, hi.w, lo.w);
            const uint32_t to = tile_piece<kPlane>(r, part * kChunks + i);
            *reinterpret_cast<uint4 *>(area + to) = hi;
            *reinterpret_cast<uint4 *>(area + kPlane * D * 2 + to) = lo;
        }
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(a.q) + at;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint4 w = live ? __ldg(reinterpret_cast<const uint4 *>(q) + i) : make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4 *>(area + tile_piece<kPlane>(r, part * kChunks + i)) = w;
        }
    }
}

// One stay on an item by the computing warps.  place0: the ring place of its first tile.
// Returns which of the item's rows (of the warp's 16, by bits) hold a value that is not
// finite.
template <int D, int MODE, int RW>
__device__ __forceinline__ unsigned rows_stay(const PagedArgs &a, const PagedItem &it, int kt0, int kt1, int part, RowsShared &sh,
                                          uint8_t *stages, uint8_t *area, uint32_t place0) {
    // Parts of the keys; TG groups of them have the tiles in turn, KW parts of KK keys each.
    // A tile of 64 columns arrives in the time that a warp's chain of waits, MMAs and softmax
    // takes, so two are worked on at once there (64 tokens of 8 kv heads over 2048 keys:
    // 70 -> 61 us, 32 rows 87 -> 81).
    constexpr int TG = D == 64 && RW <= 2 ? 2 : 1, PARTS = kRowsWarps / RW, KW = PARTS / TG, KK = kTileKeys / KW;
    constexpr int kStages = rows_stages<D>();
    // A group may wait for a stage whose use before belongs to the other group; a barrier
    // tells two phases apart, so both uses have to be the same group's.
    static_assert(TG == 1 || kStages / 2 % TG == 0, "stages and groups");
    constexpr bool F32 = MODE == PAGED_F32;
    constexpr float kScale = rows_weight_scale<MODE>();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3, mi = lane >> 3, r8 = lane & 7;
    const int rw = warp % RW, kp = warp / RW, kw = kp % KW, group = kp / KW;
    rows_load_q<D, MODE>(a, it, area, sh);
    rows_meet();
    const bool live = it.r0 + rw * 16 < it.r1;
    // Q fragments stay in registers where there is room for them beside S and O
    constexpr bool kHold = !F32 && KK <= 32;
    uint32_t q[kHold ? D / 16 : 1][4];
    const int q_at = rw * 16 + (mi & 1) * 8 + r8;
    if (kHold)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) ldmatrix_x4(q[kHold ? d : 0], area + tile_piece<kPlane>(q_at, 2 * d + (mi >> 1)));
    float fold[2];
    int lo[2], hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int lr = rw * 16 + g + 8 * r;
        paged_row_range(a, it, it.r0 + lr, lo[r], hi[r]);
        fold[r] = F32 && live ? sh.fold[lr] : a.scale_log2;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;

    for (int kt = kt0 + group; kt < kt1; kt += TG) {
        const uint32_t pk = place0 + 2 * (kt - kt0), pv = pk + 1, sk = pk % kStages, sv = pv % kStages;
        const uint8_t *ks = stages + sk * tile_bytes<D>();
        uint8_t *vs = stages + sv * tile_bytes<D>();
        const int key0 = kt * kTileKeys + kw * KK;
        float s[KK / 8][4];
        tile_wait(sh.ring, &sh.ring.full[sk], pk / kStages);
        // a warp without a row, or whose keys nobody sees, only releases the stages
        const bool busy = live && key0 < it.hi && key0 + KK > it.lo;
        if (busy) {
#pragma unroll
            for (int n = 0; n < KK / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                uint32_t x0[4], x1[4], y0[4], y1[4];
                if (kHold) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x0[i] = q[kHold ? 2 * d : 0][i];
                        x1[i] = q[kHold ? 2 * d + 1 : 0][i];
                    }
                } else {
                    ldmatrix_x4(x0, area + tile_piece<kPlane>(q_at, 4 * d + (mi >> 1)));
                    ldmatrix_x4(x1, area + tile_piece<kPlane>(q_at, 4 * d + 2 + (mi >> 1)));
                    if (F32) {
                        ldmatrix_x4(y0, area + kPlane * D * 2 + tile_piece<kPlane>(q_at, 4 * d + (mi >> 1)));
                        ldmatrix_x4(y1, area + kPlane * D * 2 + tile_piece<kPlane>(q_at, 4 * d + 2 + (mi >> 1)));
                    }
                }
#pragma unroll
                for (int n = 0; n < KK / 8; ++n) {
                    uint32_t b[4];
                    ldmatrix_x4(b, ks + tile_piece<kTileKeys>(kw * KK + n * 8 + r8, d * 4 + mi));
                    mma16<MODE>(s[n], x0, b[0], b[1]);
                    mma16<MODE>(s[n], x1, b[2], b[3]);
                    if (F32) {
                        mma16<MODE>(s[n], y0, b[0], b[1]);
                        mma16<MODE>(s[n], y1, b[2], b[3]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) tile_arrive(&sh.ring.empty[sk], TG);
        float back[2] = {1.0f, 1.0f};
        if (busy) {
            const bool whole = key0 >= it.lo_all && key0 + KK <= it.hi_all;
            float top[2] = {m[0], m[1]};
#pragma unroll
            for (int n = 0; n < KK / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i >> 1, key = key0 + 2 * t + n * 8 + (i & 1);
                    float x = s[n][i] * fold[r];
                    if (!whole && (key < lo[r] || key >= hi[r])) x = -INFINITY;
                    s[n][i] = x;
                    top[r] = fmaxf(top[r], x);
                }
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
        }
        tile_wait(sh.ring, &sh.ring.full[sv], pv / kStages);
        if (busy) {
            // keys that no row sees may hold anything: zeros, so that 0 x row stays 0
            if (key0 < it.lo || key0 + KK > it.hi) {
                for (int i = lane; i < KK * (D / 8); i += 32) {
                    const int r = i / (D / 8);
                    if (key0 + r < it.lo || key0 + r >= it.hi)
                        *reinterpret_cast<uint4 *>(vs + tile_piece<kTileKeys>(kw * KK + r, i % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();  // before the stage is loaded again
                __syncwarp();
            }
            uint32_t ph[KK / 16][4], pl[F32 ? KK / 16 : 1][4];
#pragma unroll
            for (int k = 0; k < KK / 16; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = s[2 * k + (j >> 1)][2 * (j & 1)] * kScale;
                    const float y = s[2 * k + (j >> 1)][2 * (j & 1) + 1] * kScale;
                    if (F32)
                        split_half2(x, y, ph[k][j], pl[F32 ? k : 0][j]);
                    else
                        ph[k][j] = pack2<MODE>(x, y);
                }
            if (!F32 && __any_sync(0xffffffffu, back[0] != 1.0f || back[1] != 1.0f)) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][i] *= back[i >> 1];
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                // fp32 rows: the products of a tile are summed apart and then added to O, which
                // rounds to nearest (the MMA's accumulator does not, and drifts over many tiles)
                float acc[2][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0.0f;
#pragma unroll
                for (int k = 0; k < KK / 16; ++k) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, vs + tile_piece<kTileKeys>(kw * KK + k * 16 + (mi & 1) * 8 + r8, n * 2 + (mi >> 1)));
                    mma16<MODE>(F32 ? acc[0] : o[2 * n], ph[k], b[0], b[1]);
                    mma16<MODE>(F32 ? acc[1] : o[2 * n + 1], ph[k], b[2], b[3]);
                    if (F32) {
                        mma16<MODE>(acc[0], pl[F32 ? k : 0], b[0], b[1]);
                        mma16<MODE>(acc[1], pl[F32 ? k : 0], b[2], b[3]);
                    }
                }
                if (F32)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[2 * n][i] = fmaf(o[2 * n][i], back[i >> 1], acc[0][i]);
                        o[2 * n + 1][i] = fmaf(o[2 * n + 1][i], back[i >> 1], acc[1][i]);
                    }
            }
        }
        __syncwarp();
        if (lane == 0) tile_arrive(&sh.ring.empty[sv], TG);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    if (MODE != PAGED_BF16)
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= 1.0f / kScale;
    // the key parts halve until one is left: the upper half hands its state to the lower
#pragma unroll
    for (int half = PARTS / 2; half >= 1; half >>= 1) {
        rows_meet();  // the area is free: of Q, or of what the last step left
        const int from = (kp >= half ? kp - half : kp) * RW + rw;  // 0 .. 3
        float *w = reinterpret_cast<float *>(area) + from * 32 * (D / 2) + lane;
        float2 *ml = reinterpret_cast<float2 *>(area + 4 * 32 * (D / 2) * 4) + from * 16 + g;
        if (kp >= half && kp < 2 * half && live) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[(n * 4 + i) * 32] = o[n][i];
            if (t == 0) {
                ml[0] = make_float2(m[0], l[0]);
                ml[8] = make_float2(m[1], l[1]);
            }
        }
        rows_meet();
        if (kp < half && live) {
            float mine[2], other[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float2 x = ml[8 * r];
                const float mx = fmaxf(m[r], x.x), base = mx == -INFINITY ? 0.0f : mx;
                mine[r] = exp2_fast(m[r] - base);
                other[r] = exp2_fast(x.x - base);
                l[r] = l[r] * mine[r] + x.y * other[r];
                m[r] = mx;
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][i] = o[n][i] * mine[i >> 1] + w[(n * 4 + i) * 32] * other[i >> 1];
        }
    }
    unsigned odd_rows = 0;
    if (kp == 0 && live) {
        bool odd[2] = {false, false};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = it.r0 + rw * 16 + g + 8 * r;
            if (row >= it.r1) continue;
            if (part >= 0) {
                const int64_t at = static_cast<int64_t>(part) * a.item_rows + row - it.r0;
                float *po = a.parts[0].o + at * D;
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2 *>(po + n * 8 + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if (t == 0) *reinterpret_cast<float2 *>(a.parts[0].ml + at * 2) = make_float2(m[r], l[r]);
                continue;
            }
            const float inv = 1.0f / l[r];
            const int64_t at = paged_row_offset(a, it, row, a.out_row, D);
            float probe = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                const float x = o[n][2 * r] * inv, y = o[n][2 * r + 1] * inv;
                probe += 0.0f * x + 0.0f * y;
                if (F32)
                    *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + n * 8 + 2 * t) = make_float2(x, y);
                else
                    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at + n * 8 + 2 * t) =
                        pack2<MODE>(paged_bounded<MODE>(x), paged_bounded<MODE>(y));
            }
            odd[r] = !(probe == 0.0f);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const unsigned vote = __ballot_sync(0xffffffffu, odd[r]);
#pragma unroll
            for (int x = 0; x < 8; ++x) odd_rows |= (vote >> (4 * x) & 0xF) ? 1u << (x + 8 * r) : 0u;
        }
    }
    return odd_rows;
}

template <int D, int MODE>
__global__ void __launch_bounds__(kRowsThreads, 1)
    paged_rows_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      int heads_outer) {
    constexpr int kStages = rows_stages<D>();
    extern __shared__ uint8_t rows_raw[];
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rows_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *area = stages + kStages * tile_bytes<D>();
    __shared__ RowsShared sh;
    const int tid = threadIdx.x, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.ring.full[s], 1);
            mbar_init(&sh.ring.empty[s], kRowsWarps);
        }
        sh.ring.abort = sh.ring.slow = 0;
        mbar_init_fence();
    }
    __syncthreads();
    grid_wait();
    grid_launch_dependents();
    constexpr int M = rows_item(D, MODE);
    PagedWalk<M, kTileKeys, rows_extra<D, MODE>(), false> walk;
    if (tid == 0) a.parts[0].open[blockIdx.x].last = -1;
    if (!walk.begin(a, sh.walk, blockIdx.x, gridDim.x)) return;
    // registers: 384 x 168 at launch = 128 x 56 + 256 x 224
    if (warp >= kRowsWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        load_tiles<D, kStages, 4>(a, walk, sh.ring, stages, &k_map, &v_map, heads_outer, -1, warp - kRowsWarps);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        uint32_t place = 0;
        PagedItem it;
        int kt0, kt1, part;
        while (walk.next(a, it, kt0, kt1, part)) {
            const int rows = it.r1 - it.r0;
            if (tid == 0 && part >= 0 && (part & 1)) a.parts[0].open[blockIdx.x] = PagedOpen{it, walk.last_cta()};
            unsigned odd;
            int row0;  // of the warp
            // (what an item's size does not need is not in the kernel: more code costs 8 %)
            if (M == 16 || rows <= 16) {
                odd = rows_stay<D, MODE, 1>(a, it, kt0, kt1, part, sh, stages, area, place);
                row0 = 0;
            } else if (M == 32 || rows <= 32) {
                odd = rows_stay<D, MODE, M >= 32 ? 2 : 1>(a, it, kt0, kt1, part, sh, stages, area, place);
                row0 = warp % 2 * 16;
            } else {
                odd = rows_stay<D, MODE, M >= 64 ? 4 : 1>(a, it, kt0, kt1, part, sh, stages, area, place);
                row0 = warp % 4 * 16;
            }
            // rows with a value that is not finite are done again, key by key
            __syncwarp();
            slow_rows<D, MODE>(a, it, sh.ring, it.r0 + row0, odd);
            rows_meet();  // the area is free for the next Q
            place += 2 * (kt1 - kt0);
        }
        if (sh.ring.abort && tid == 0) set_flag(a.flags, BD_FLAG_TIMEOUT);
    }
}

template <int D, int MODE>
static int launch_rows(const PagedArgs &a, const PagedMaps &maps, int ctas, cudaStream_t stream) {
    auto kernel = paged_rows_kernel<D, MODE>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(rows_smem<D>())) != cudaSuccess)
        return BD_ERR_LAUNCH;
    return launch_pdl(kernel, dim3(ctas), dim3(kRowsThreads), rows_smem<D>(), stream, a, maps.k, maps.v, maps.heads_outer);
}

int launch_paged_rows(const PagedArgs &a, const PagedMaps &maps, int head_dim, int mode, int ctas, cudaStream_t stream) {
    if (head_dim == 64)
        return mode == PAGED_F32   ? launch_rows<64, PAGED_F32>(a, maps, ctas, stream)
               : mode == PAGED_F16 ? launch_rows<64, PAGED_F16>(a, maps, ctas, stream)
                                   : launch_rows<64, PAGED_BF16>(a, maps, ctas, stream);
    return mode == PAGED_F32   ? launch_rows<128, PAGED_F32>(a, maps, ctas, stream)
           : mode == PAGED_F16 ? launch_rows<128, PAGED_F16>(a, maps, ctas, stream)
                               : launch_rows<128, PAGED_BF16>(a, maps, ctas, stream);
}

}  // namespace bd
