// Attention over the paged cache on the 5th-generation tensor cores (tcgen05, TMEM), for
// fp16 and bf16 rows.  The mathematics, the item / unit / range split and the joining
// of partials are those of paged_attention.cu, with 256 rows to an item.  (fp32 rows,
// as hi and lo halves of Q and P, ran here 14 % faster at 24 blocks of 64 rows, but the
// accumulators in TMEM truncate: 3.9e-6 off after 2000 keys against 1e-6 there.)
//
// One CTA per SM.  Two streams of work alternate on the tensor pipe:
//   * an item of more than 128 rows: stream t has rows [128 t, 128 t + 128), and both
//     use every key tile, which is loaded once;
//   * an item of up to 128 rows: both streams have the same rows, stream t takes keys
//     [64 t, 64 t + 64) of every tile, and the two (maximum, sum, O) are joined at the
//     end of the stay.
// A stream goes by steps of 64 keys and has two buffers for S, so that its next S is
// ready when the softmax of this one ends: with one buffer of 128 keys the chain S,
// softmax, P V of a stream left the tensor pipe 55 % idle (8192 + 2048 keys: 681 us).
// Warps 0-3 and 4-7 are the softmax of stream 0 and 1, a thread to a row: S from
// TMEM, running maximum and sum, P as 16-bit values back over S's columns.  O stays
// in TMEM; a row's O is rescaled only when its maximum has grown by more than 2^8 (fp16
// rows 2^4) since the last time (the sum and O scale alike), which takes the rescaling off the
// usual path.  Warps 10 and 11 load key and value tiles by TMA
// (a box per page piece and 64 columns) into one ring in the order of their use;
// warps 8 and 9 issue, each for a stream, S = Q K^T (both operands in shared memory)
// and O += P V (P in TMEM, V as it lies, its rows being the reduction).
//
// What bounds it: in the steady state the softmax's chain of a step (two 2048-token chunks
// over 8192 more keys: 575 us = 1075 TFLOP/s, at the GPU's power limit 650; with the softmax left out it would be 1350),
// and some 10,000 cycles a stay for Q, the first products and the output (over 4096 more
// keys 340 us = 1010 TFLOP/s, ragged chunks of 64 columns in a window of 1000 keys 51 us).
// Verification (32 requests of 68 rows over 0.5 to 4 K keys) takes 62 us = 4.5 TB/s.
//
// Every wait is bounded; one that runs out sets BD_FLAG_TIMEOUT and turns the waits
// that follow into passes, so that all roles walk to their end.
#include "paged_attention.cuh"

namespace bd {

constexpr int kTcStep = 64;  // keys of a step of a stream
constexpr int kTcThreads = 384;
// A stay's Q, first and last products and output, in units: 3 to 4 where a tile has 256 rows, 6
// to 8 with up to 128 (32 x 17 ragged tokens: 76 us with 3, 74 with 4, 69 with 6, 73 with 8; two
// 2048-token chunks 244, 235, 234 and 247).
constexpr int kTcExtra = 6;
// A row's weights are 2^(x - base), with the base kTcShift below its maximum as it was at the last
// rescaling; growth of the maximum by up to kTcSlack leaves base and O as they are.  For fp16
// the two add up to 2^15, so that weights down to 2^-36 of the largest are held (with a shift of
// 0 and a slack of 8, those under 2^-25 were lost to O and not to the sum); bf16 has fp32's range.
template <int MODE>
constexpr float tc_shift() {
    return MODE == PAGED_F16 ? 11.0f : 0.0f;
}
template <int MODE>
constexpr float tc_slack() {
    return MODE == PAGED_F16 ? 4.0f : 8.0f;
}
// The base of a maximum; from 2^20 on, where its own steps are larger than a sixteenth, without the shift.
template <int MODE>
__device__ __forceinline__ float tc_base(float m) {
    return m == -INFINITY ? 0.0f : (fabsf(m) < 1048576.0f ? m - tc_shift<MODE>() : m);
}

template <int D>
constexpr int tc_stages() {
    return D == 128 ? 5 : 8;
}
template <int D>
constexpr size_t tc_smem() {
    return 1024 + 2 * 128 * D * 2 + static_cast<size_t>(tc_stages<D>()) * tile_bytes<D>();
}

struct TcShared {
    TileRing ring;
    // of a stream and of its S buffers.  A barrier's wait tells two phases apart, no more:
    // o_step is for the products of a step, o_full for those of a stay.
    uint64_t q_full, s_full[2][2], p_full[2][2], o_step[2][2], o_full[2], drain[2];
    uint32_t tmem;
    float2 ml[128];
    PagedShared walk;
};

__device__ __forceinline__ void tc_commit(uint64_t *b, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(b)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 lanes x 32 columns of TMEM: lane = row, register = column.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
        "%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// 16 columns, for the loops beside the main one (rolled: their code is fetched anew at
// every stay).
__device__ __forceinline__ void tc_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operands are 128-byte-swizzled rows of 64 values; a tile of D
// columns is D / 64 such blocks of 128 rows (16 KB) one behind the other.  The lower
// word of a matrix descriptor is the address and the leading offset, the upper one is
// the same for all: 8-row groups 1024 B apart, 128-byte swizzle.
// K-major (Q, K): a step of 16 columns is 32 B; the leading offset is not used.
// MN-major (V, whose rows are the reduction): 64-column blocks 16 KB apart, a step of
// 16 rows is 2 KB.
constexpr uint32_t kTcDescUpper = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc_desc_rows(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t tc_desc_cols(uint32_t addr) { return (addr >> 4) | ((16384u >> 4) << 16); }
// kind::f16 instruction descriptor: fp32 accumulators, M = 128, A and B fp16 or bf16.
__host__ __device__ constexpr uint32_t tc_idesc(bool bf16, int n, bool b_cols) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_cols ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}
// One MMA, issued by the lane whose `leader` is set.  The whole warp runs the code
// around it, so that its operands can be warp-uniform registers.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.u32 p, %5, 0;\n setp.ne.u32 q, %6, 0;\n"
        " mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(kTcDescUpper), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 b;\n setp.ne.u32 p, %5, 0;\n setp.ne.u32 q, %6, 0;\n"
        " mov.b64 b, {%2, %3};\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(kTcDescUpper), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ uint32_t tc_elect() {
    uint32_t leader;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(leader));
    return leader;
}
// A value that is the same in all lanes, as one the compiler knows to be: a reduction
// over the warp leaves its result in a uniform register.
__device__ __forceinline__ uint32_t tc_uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }
__device__ __forceinline__ float max3(float x, float y, float z) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}

template <int MODE>
__device__ __forceinline__ uint32_t tc_pack(float lo, float hi) {
    if (MODE == PAGED_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The issuing warp of stream t.  A warp of its own for each stream: between two groups of
// MMAs stand waits and commits of some 600 cycles, more than the tensor pipe has
// queued, which the other stream's MMAs fill.  All that an MMA takes is warp-uniform to
// the compiler's eyes (moving operands to uniform registers took longer than the
// MMAs), and each product stands once in the code, which all roles together must
// keep small: a stay's own code is fetched anew after every main loop.
template <int D, int MODE>
struct TcIssuer {
    static constexpr int kStages = tc_stages<D>(), kStage = tile_bytes<D>();
    static constexpr bool BF16 = MODE == PAGED_BF16;
    static constexpr uint32_t kScores = tc_idesc(BF16, kTcStep, false), kValues = tc_idesc(BF16, D, true);
    static constexpr uint32_t kHalf = kTcStep * 128 >> 4;  // of a tile, in descriptor units
    TcShared &sh;
    uint8_t *ring;
    const uint32_t t;
    uint32_t s_columns, o_columns, q_desc, k_desc, v_desc, go;
    uint32_t p_phase = 0;               // bit b: of S buffer b
    uint32_t next = 0, next_phase = 0;  // the ring's next tile, in the order of first use
    uint32_t k_stage = 0, v_stage = 0;  // the tiles in use

    __device__ __forceinline__ TcIssuer(TcShared &s, uint32_t q, uint8_t *r, uint32_t stream) : sh(s), ring(r), t(stream) {
        s_columns = tc_uniform(s.tmem) + t * 128;
        o_columns = s_columns + 256;
        q_desc = tc_desc_rows(q);
        k_desc = tc_desc_rows(smem_u32(r));
        v_desc = tc_desc_cols(smem_u32(r));
        go = tc_elect();
    }
    __device__ __forceinline__ void wait(uint64_t *b, uint32_t count) {
        if (!warp_wait(sh.ring, b, count)) go = 0;
        tc_fence_after();
    }
    __device__ __forceinline__ void tile(uint32_t &stage) {
        stage = next;
        wait(&sh.ring.full[stage], next_phase);
        next = next + 1 == kStages ? 0 : next + 1;
        next_phase ^= next == 0;
    }
    // The products of a stay of n key tiles: before O += P V of step i, whose 64 keys are half
    // i & 1 of a tile, or with the same rows in both streams half t of tile i, stands S = Q K^T
    // of steps i and i + 1.
    __device__ __forceinline__ void stay(const PagedItem &it, int kt0, int n, bool both) {
        const int steps = both ? 2 * n : n;
        const uint32_t q0 = q_desc + (both ? t * (128 * D * 2 >> 4) : 0);
#pragma unroll 1
        for (int i = -2; i < steps; ++i) {
            const uint32_t b = i & 1, half = both ? b : t;
            const bool first = !both || b == 0, last = !both || b == 1;  // use of a tile
            if (i >= 0) {
                if (first) {
                    tile(v_stage);
                    // rows of keys that no row sees may hold anything: zeros, so that 0 x row stays 0
                    // (both streams' warps write them, each before its own products)
                    const int key0 = (kt0 + (both ? i >> 1 : i)) * kTileKeys;
                    if (tc_uniform(key0 < it.lo || key0 + kTileKeys > it.hi)) {
                        for (int x = threadIdx.x & 31; x < kTileKeys * (D / 8); x += 32) {
                            const int r = (x >> 3) & (kTileKeys - 1);
                            if (key0 + r < it.lo || key0 + r >= it.hi)
                                *reinterpret_cast<uint4 *>(ring + v_stage * kStage + x * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                wait(&sh.p_full[t][b], p_phase >> b);
                const uint32_t v0 = v_desc + v_stage * (kStage >> 4) + half * kHalf, from = s_columns + b * kTcStep;
#pragma unroll
                for (int k = 0; k < kTcStep / 16; ++k)
                    tc_mma_ts(o_columns, from + k * 8, v0 + k * (2048 >> 4), kValues, k > 0 ? 1u : i > 0, go);
                tc_commit(&sh.o_step[t][b], go);
                if (last) tc_commit(&sh.ring.empty[v_stage], go);
                p_phase ^= 1u << b;
            }
            if (i + 2 < steps) {
                if (first) tile(k_stage);
                const uint32_t k0 = k_desc + k_stage * (kStage >> 4) + half * kHalf, to = s_columns + b * kTcStep;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                    tc_mma_ss(to, q0 + at, k0 + at, kScores, k > 0, go);
                }
                tc_commit(&sh.s_full[t][b], go);
                if (last) tc_commit(&sh.ring.empty[k_stage], go);
            }
        }
        tc_commit(&sh.o_full[t], go);
    }
    template <typename Walk>
    __device__ __forceinline__ void run(const PagedArgs &a, Walk &walk) {
        uint32_t stays = 0;
        PagedItem it;
        int kt0, kt1, out;
        while (tc_uniform(walk.next(a, it, kt0, kt1, out))) {
            wait(&sh.q_full, stays++);
            stay(it, kt0, tc_uniform(kt1 - kt0), tc_uniform(it.r1 - it.r0 > 128));
        }
        // every product issued completes before TMEM is freed
        tc_commit(&sh.drain[t], tc_elect());
        mbar_wait_bounded(&sh.drain[t], 0, kTilePolls);
    }
};

template <int D, int MODE>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_tc_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                    int heads_outer) {
    constexpr int kStages = tc_stages<D>();
    constexpr uint32_t kO = 256;  // TMEM columns: two S buffers of each stream (P over them), O at 256 and 384
    extern __shared__ uint8_t tc_raw[];
    uint8_t *sq = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = sq + 2 * 128 * D * 2;
    __shared__ TcShared sh;
    const int tid = threadIdx.x, warp = static_cast<int>(tc_uniform(tid >> 5)), lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.ring.full[s], 1);
            mbar_init(&sh.ring.empty[s], 2);
        }
        mbar_init(&sh.q_full, 8);
        for (int t = 0; t < 2; ++t) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.s_full[t][i], 1);
                mbar_init(&sh.p_full[t][i], 4);
                mbar_init(&sh.o_step[t][i], 1);
            }
            mbar_init(&sh.o_full[t], 1);
            mbar_init(&sh.drain[t], 1);
        }
        sh.ring.abort = sh.ring.slow = 0;
        mbar_init_fence();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    grid_wait();
    grid_launch_dependents();
    PagedWalk<kTcItem, kTileKeys, kTcExtra, true> walk;
    if (tid == 0) a.parts[1].open[blockIdx.x].last = -1;
    const bool any = walk.begin(a, sh.walk, blockIdx.x, gridDim.x);
    // registers: 384 x 168 at launch = 128 x 104 + 256 x 200
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (any && warp < 10)
            TcIssuer<D, MODE>(sh, smem_u32(sq), ring, warp - 8).run(a, walk);
        else if (any)
            load_tiles<D, kStages, 2>(a, walk, sh.ring, ring, &k_map, &v_map, heads_outer, 128, warp - 10);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // -------------------------------------------------- softmax: a thread to a row
        const int t = warp >> 2, wrow = (warp & 3) * 32, lrow = wrow + lane;
        const uint32_t s_at = tmem + t * 128 + (static_cast<uint32_t>(wrow) << 16), o_at = s_at + kO;
        // the scale's sign goes into Q; not 0, as a masked -inf times it has to stay that (the smallest
        // number there is, 2^-149, leaves every finite score at 0)
        const float c = fmaxf(fabsf(a.scale_log2), 1.4e-45f);
        // 16-byte piece c of row r of 128 rows as the MMAs read them
        auto row_piece = [](uint8_t *rows, int r, int c) {
            return reinterpret_cast<uint4 *>(rows + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
        };
        constexpr int kLanes = D / 8, kPass = 32 / kLanes;  // lanes to a row of D 16-bit values, rows of a warp's access
        const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
        uint32_t steps[2] = {0, 0}, stays = 0;  // steps: through each S buffer
        PagedItem it;
        int kt0, kt1, out;
        while (any && walk.next(a, it, kt0, kt1, out)) {
            const int n = kt1 - kt0, rows = it.r1 - it.r0;
            if (tid == 0 && out >= 0 && (out & 1)) a.parts[1].open[blockIdx.x] = PagedOpen{it, walk.last_cta()};
            const bool both = rows > 128;
            const int count = both ? 2 * n : n;  // steps of 64 keys
            const int row = it.r0 + (both ? t * 128 : 0) + lrow;
            const bool live = row < it.r1;
            const bool warp_live = row - lane < it.r1;
            int lo, hi;
            paged_row_range(a, it, row, lo, hi);
            // Q rows into shared memory, whole rows by neighbouring lanes: a warp's own 32, or 16
            // of those that both streams have
            if (!both) asm volatile("bar.sync 1, 256;" ::: "memory");  // both streams have left the last stay
            uint8_t *rows_at = sq + (both ? t * 128 * D * 2 : 0);
            {
                const int first = (both ? wrow : warp * 16) + lane / kLanes, c = lane % kLanes;
                const int row0 = it.r0 + (both ? t * 128 : 0);
                const int end = both ? 32 : 16;
#pragma unroll 1
                for (int i0 = 0; i0 < end; i0 += 8 * kPass) {
                    uint4 w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = row0 + first + i0 + i * kPass;
                        w[i] = make_uint4(0u, 0u, 0u, 0u);
                        if (r < it.r1)
                            w[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) +
                                                                         paged_row_offset(a, it, r, a.q_row, a.q_head)) + c);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *row_piece(rows_at, first + i0 + i * kPass, c) =
                            make_uint4(w[i].x ^ flip, w[i].y ^ flip, w[i].z ^ flip, w[i].w ^ flip);
                }
            }
            fence_proxy_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) tile_arrive(&sh.q_full);

            float m = -INFINITY, base = 0.0f, l = 0.0f;
            for (int i = 0; i < count; ++i) {
                const int buffer = i & 1;
                const uint32_t at = s_at + buffer * kTcStep;
                tile_wait(sh.ring, &sh.s_full[t][buffer], steps[buffer]++);
                tc_fence_after();
                if (warp_live) {
                    const int key0 = both ? (kt0 * 2 + i) * kTcStep : (kt0 + i) * kTileKeys + t * kTcStep;
                    float s[2][32];
                    tc_ld32(at, s[0]);
                    tc_ld32(at + 32, s[1]);
                    tc_ld_wait();
                    if (key0 < it.lo_all || key0 + kTcStep > it.hi_all) {
                        const int first = lo - key0, last = hi - key0;
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (32 * x + k < first || 32 * x + k >= last) s[x][k] = -INFINITY;
                    }
                    float top[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float *v = &s[x >> 1][(x & 1) * 16];
                        top[x] = fmaxf(v[0], v[1]);
#pragma unroll
                        for (int k = 2; k < 16; k += 2) top[x] = max3(top[x], v[k], v[k + 1]);
                    }
                    const float now = fmaxf(max3(top[0], top[1], top[2]), top[3]) * c;
                    const bool grows = now > m + tc_slack<MODE>() || m == -INFINITY;
                    if (__any_sync(0xffffffffu, grows && m != -INFINITY)) {
                        // the products so far are in O (this S says so of all but the last step's)
                        tile_wait(sh.ring, &sh.o_step[t][buffer ^ 1], steps[buffer ^ 1] - 1);
                        tc_fence_after();
                        const float back = grows ? exp2_fast(base - tc_base<MODE>(now)) : 1.0f;
                        l *= m == -INFINITY ? 1.0f : back;
#pragma unroll 1
                        for (int x = 0; x < D / 16; ++x) {
                            float o[16];
                            tc_ld16(o_at + 16 * x, o);
                            tc_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = m == -INFINITY ? 0.0f : o[k] * back;
                            tc_st16(o_at + 16 * x, o);
                        }
                    }
                    if (grows) {
                        m = now;
                        base = tc_base<MODE>(now);
                    }
                    const float2 c2 = make_float2(c, c), base2 = make_float2(-base, -base);
                    float2 sum[4];
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float *x = &s[k >> 4][2 * (k & 15)];
                        float2 p = __ffma2_rn(make_float2(x[0], x[1]), c2, base2);
                        p = make_float2(exp2_fast(p.x), exp2_fast(p.y));
                        sum[k & 3] = k < 4 ? p : __fadd2_rn(sum[k & 3], p);
                        w[k] = tc_pack<MODE>(p.x, p.y);
                    }
                    tc_st32(at, w);
                    const float2 all = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
                    l += all.x + all.y;
                    tc_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tile_arrive(&sh.p_full[t][buffer]);
            }
            tile_wait(sh.ring, &sh.o_full[t], stays++);
            tc_fence_after();
            if (m != -INFINITY) m = base;  // what l and O are relative to
            float4 *swap = reinterpret_cast<float4 *>(sq);  // Q is done with: O of stream 1, [column / 4][row]
            float mine_w = 1.0f, other_w = 0.0f;
            if (!both) {
                asm volatile("bar.sync 1, 256;" ::: "memory");  // neither stream reads Q any more
                if (t == 1 && warp_live) {
                    sh.ml[lrow] = make_float2(m, l);
#pragma unroll 1
                    for (int i = 0; i < D / 16; ++i) {
                            float o[16];
                            tc_ld16(o_at + 16 * i, o);
                            tc_ld_wait();
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                swap[(i * 4 + k) * 128 + lrow] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                        }
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (t == 0 && warp_live) {
                    const float2 x = sh.ml[lrow];
                    const float top = fmaxf(m, x.x);
                    base = top == -INFINITY ? 0.0f : top;
                    mine_w = exp2_fast(m - base);
                    other_w = exp2_fast(x.x - base);
                    l = l * mine_w + x.y * other_w;
                    m = top;
                }
            }
            if ((both || t == 0) && warp_live) {
                const float inv = out >= 0 ? 1.0f : 1.0f / l;
                float probe = 0.0f;
                const int64_t part_row = static_cast<int64_t>(max(out, 0)) * kTcItem + row - it.r0;
                const int64_t at = live ? paged_row_offset(a, it, row, a.out_row, D) : 0;
                // a row's 16 columns from TMEM go to memory from here when the rows are few; else by way
                // of the warp's Q rows (done with), so that neighbouring lanes store whole rows: all
                // 16-bit columns at once, partials in two halves
                const int passes = out >= 0 ? 2 : 1, each = D / 16 / passes;
                for (int pass = 0; pass < passes; ++pass) {
#pragma unroll 1
                    for (int i = pass * each; i < (pass + 1) * each; ++i) {
                        float o[16];
                        tc_ld16(o_at + 16 * i, o);
                        tc_ld_wait();
                        if (!both) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float4 x = swap[(i * 4 + k) * 128 + lrow];
                                o[4 * k] = o[4 * k] * mine_w + x.x * other_w;
                                o[4 * k + 1] = o[4 * k + 1] * mine_w + x.y * other_w;
                                o[4 * k + 2] = o[4 * k + 2] * mine_w + x.z * other_w;
                                o[4 * k + 3] = o[4 * k + 3] * mine_w + x.w * other_w;
                            }
                        }
                        if (out >= 0) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float4 x = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                                if (both)
                                    *reinterpret_cast<float4 *>(row_piece(rows_at, lrow, (i - pass * each) * 4 + k)) = x;
                                else if (live)
                                    *reinterpret_cast<float4 *>(a.parts[1].o + part_row * D + 16 * i + 4 * k) = x;
                            }
                        } else {
                            uint32_t w[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float x = o[2 * k] * inv, y = o[2 * k + 1] * inv;
                                probe += 0.0f * x + 0.0f * y;
                                w[k] = tc_pack<MODE>(paged_bounded<MODE>(x), paged_bounded<MODE>(y));
                            }
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint4 x = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                                if (both)
                                    *row_piece(rows_at, lrow, 2 * i + k) = x;
                                else if (live)
                                    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + at + 16 * i + 8 * k) = x;
                            }
                        }
                        __syncwarp();
                    }
                    if (both) {
#pragma unroll 2
                        for (int i = 0; i < 32; i += kPass) {
                            const int lr = wrow + i + lane / kLanes, c = lane % kLanes, r = it.r0 + t * 128 + lr;
                            if (r >= it.r1) continue;
                            const uint4 x = *row_piece(rows_at, lr, c);
                            if (out >= 0)
                                reinterpret_cast<uint4 *>(a.parts[1].o + (static_cast<int64_t>(out) * kTcItem + r - it.r0) * D +
                                                          pass * (D / 2))[c] = x;
                            else
                                reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) +
                                                          paged_row_offset(a, it, r, a.out_row, D))[c] = x;
                        }
                        __syncwarp();
                    }
                }
                if (out >= 0 && live) *reinterpret_cast<float2 *>(a.parts[1].ml + part_row * 2) = make_float2(m, l);
                // rows with a value that is not finite are done again, key by key
                slow_rows<D, MODE>(a, it, sh.ring, row - lane, __ballot_sync(0xffffffffu, live && out < 0 && !(probe == 0.0f)));
            }
            tc_fence_before();
            if (!both) asm volatile("bar.sync 1, 256;" ::: "memory");  // the swap area is free
        }
    }
    if (sh.ring.abort && tid == 0) set_flag(a.flags, BD_FLAG_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
    }
}

static_assert(tc_smem<128>() + sizeof(TcShared) + 16 <= 232448 && tc_smem<64>() + sizeof(TcShared) + 16 <= 232448,
              "one CTA's shared memory");

template <int D, int MODE>
static int launch_tc(const PagedArgs &a, const PagedMaps &maps, int ctas, cudaStream_t stream) {
    if (cudaFuncSetAttribute(paged_tc_kernel<D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(tc_smem<D>())) != cudaSuccess)
        return BD_ERR_LAUNCH;
    return launch_pdl(paged_tc_kernel<D, MODE>, dim3(ctas), dim3(kTcThreads), tc_smem<D>(), stream, a, maps.k, maps.v,
                      maps.heads_outer);
}

int launch_paged_tc(const PagedArgs &a, const PagedMaps &maps, int head_dim, int mode, int ctas, cudaStream_t stream) {
    if (head_dim == 64)
        return mode == PAGED_F16 ? launch_tc<64, PAGED_F16>(a, maps, ctas, stream)
                                 : launch_tc<64, PAGED_BF16>(a, maps, ctas, stream);
    return mode == PAGED_F16 ? launch_tc<128, PAGED_F16>(a, maps, ctas, stream)
                             : launch_tc<128, PAGED_BF16>(a, maps, ctas, stream);
}

}  // namespace bd
