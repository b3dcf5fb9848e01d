// Products of many rows over weights held in 4 bits (the format: quant4.cuh), on the 5th-generation tensor cores.
//
// A warp takes the codes of a strip (16 features x 64 k) as they lie in global memory, forms the bfloat16 values q s (exact) in registers and writes
// them to the stage's tile in shared memory (rows of 128 bytes, the swizzle that TMA would have given them; odd rows write their 16-byte pieces in
// another order, so that no two lanes meet in a bank).  The rows of x come by TMA.  Two accumulators (all 512 columns of tensor memory), so the epilogue
// of a tile runs under the next one's products.  A tile is
//
//   narrow   128 features, the MMA's lanes (A), x up to 256 rows, its columns (B)
//   wide     256 features, its columns, x 128 rows, its lanes: for groups of few rows, because an MMA of 128 lanes takes 150 cycles and more for 16 k
//            whatever its columns
//
//   2 teams   of a warp for 32 features: every second block of 64 k to values, two of its blocks ahead in registers
//   8 warps   epilogue: accumulator -> registers -> global memory (warp w: lanes 32 (w % 4).., half of the columns)
//   1 warp    TMA producer of the rows of x
//   1 warp    allocates tensor memory and issues the products
//
// What bounds a tile is shared memory's 128 bytes a cycle: 16 k of the values are written and read (narrow 64 cycles, wide 128), of the rows too (N / 2,
// 64), against N / 2 (128) cycles of the tensor core.  Measured a block of 64 k: narrow 810 cycles at 136 rows, wide 1,055 (one team: 1,443, all of
// it forming values; three teams, without registers for it, 1,070).  2,048 rows of a pair 11,264 x 2,048 83 us (1.14 PFLOP/s), 8,192 of 60 experts 146 us, 2,048 of
// them 101 us.  (With the values in tensor memory instead, tcgen05.st in the codes' own layout, a product took 128 cycles whatever N, to load A, and
// 190 beside the stores: 2,048 rows of a pair 11,264 x 2,048 113 us, 8,192 rows of 2,048 x 5,632 240 us.)
//
// One CTA an SM walks over the tiles.  A gated pair's tile holds half as many features: gate strips in rows 32 i.., up strips in rows 32 i + 16.. .
// Groups (routed experts): rows [offsets[g], offsets[g + 1]) meet the weights of g.  Where a dense product has too few tiles for the
// SMs, up to 8 CTAs of a cluster share a tile's k; each leaves its partial sums in its shared memory, and each adds up an equal share of the rows in
// the order of the splits.
//
// Every wait on a barrier is bounded; one that runs out sets ST_WAIT_TIMEOUT, the roles drain and the CTA frees its tensor memory.
#include <cuda.h>

#include <mutex>

#include "quant4.cuh"

namespace {

using q4::Weight;

constexpr int BK = 64, BN = 256, NBUF = 2, STAGES_MAX = 8;
constexpr int BOX = 64, BOX_BYTES = BOX * BK * 2, ROOM = 200 * 1024;      // ROOM: bytes for stages
constexpr int TMEM_COLS = 512, MAX_GROUPS = 1024, MAX_CLUSTER = 4;
static_assert(NBUF * BN <= TMEM_COLS, "tensor memory");
// WIDE: 256 features, the MMA's columns, x 128 rows; else 128 features, the MMA's lanes, x up to 256 rows
template <bool WIDE>
struct Form {
    static constexpr int FEATURES = WIDE ? 256 : 128, W_BYTES = FEATURES * BK * 2;
    static constexpr int TEAM = FEATURES / 32, TEAMS = 2, PREFETCH = 2;      // warps that form a block's values, 32 rows of it each
    static constexpr int DEQUANT_WARPS = TEAM * TEAMS, EPI_WARPS = 8, WARPS = DEQUANT_WARPS + EPI_WARPS + 2, THREADS = WARPS * 32;
};

struct Args {
    Weight w;
    void* out;
    int out_bf16, ldo;
    const float* bias;
    const int* offsets;
    int G, M, N;                   // N: output features
    int vec;                       // rows of the output in whole 16-byte units
    int bn;                        // rows of a tile, a multiple of 16
    int stages, stage_bytes;       // values and boxes of 64 rows
    int n_tiles;                   // tiles of features
    int splits, kb_per_split;
    int act;
    float act_param;
    int* status;
    int early;                     // the weight may be read before what is in front of this launch has ended
    uint32_t wait_limit;
    q4::Bits bits;
    int test_fault;                // 0; the wait test: 1 nothing is loaded, 2 no product is issued, 3 no value is formed
};

// ---- PTX wrappers ----------------------------------------------------------------------------------------------------------------------
using q4::mbar_arrive;
using q4::mbar_expect_tx;
using q4::mbar_init;
using q4::smem_u32;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const Args& p, int site) {
    return q4::mbar_wait(bar, parity, abort_flag, p.wait_limit, p.status, site);
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(bar)
                 : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// D[128, N] (+)= A[128, 16] B[N, 16]^T, both in shared memory
__device__ __forceinline__ void umma(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
// K-major tile with 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// 32-bit sums, bfloat16 operands, both K-major
__device__ __forceinline__ uint32_t instr_desc(int n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

struct Tile {
    int g, row0, rows, ft;         // group, first row, rows, tile of features
};
__device__ __forceinline__ Tile tile_of(int item, int m_tiles, const Args& p, const int* prefix, const int* offs) {
    Tile t;
    if (!p.offsets) {              // all row tiles of a feature tile first: CTAs that run together share its codes in L2
        t.ft = item / m_tiles, t.g = 0, t.row0 = (item % m_tiles) * p.bn, t.rows = min(p.bn, p.M - t.row0);
        return t;
    }
    const int m = item / p.n_tiles;      // all feature tiles of a row tile first: they share its rows
    t.ft = item % p.n_tiles;
    int lo = 0, hi = p.G;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= m) lo = mid; else hi = mid;
    }
    t.g = lo, t.row0 = offs[lo] + (m - prefix[lo]) * p.bn, t.rows = min(p.bn, offs[lo + 1] - t.row0);
    return t;
}

__device__ __forceinline__ void put(const Args& p, int row, int n, float v) {
    if (p.out_bf16)
        ((__nv_bfloat16*)p.out)[(size_t)row * p.ldo + n] = __float2bfloat16_rn(v);
    else
        ((float*)p.out)[(size_t)row * p.ldo + n] = v;
}

// silu(g) u by the quick exponential and quotient.  The exponential is within 2 + 1.2 |g| ulp of 32 bits, the quotient within 2 (and 0 from a divisor of 2^126 on, where silu
// is 8e-37 and less): 2^-21 at gates of order one, 2^-16 at -100, where the few-row forms' functions have 2^-20 throughout.  With those the epilogue of a prompt's tiles is
// 3 to 4 % of the product's time longer (2,048 rows of 60 experts, a pair 2,816 x 2,048: 146 -> 150 us).
__device__ __forceinline__ float gated(const Args& p, float g, float u) {
    if (p.act == ACT_SILU) return __fdividef(g, 1.f + __expf(-g)) * u;
    return glu_mul(p.act, p.act_param, g, u);
}

// Rows [lo, hi) of a finished tile by one warp: lanes 32 q.. of the accumulator at taddr
template <bool PAIR, typename T>
__device__ __forceinline__ void store_part(const Args& p, T* out, const Tile& t, uint32_t taddr, int q, int lane, int lo, int hi) {
    const bool upper = PAIR && (lane & 16);
    const int n = PAIR ? t.ft * 64 + q * 16 + (lane & 15) : t.ft * 128 + q * 32 + lane;
    const float bias = !PAIR && p.bias && n < p.N ? p.bias[n] : 0.f;
    const bool live = n < p.N;
    T* o = out + (size_t)(t.row0 + lo) * p.ldo + n;
    for (int c0 = lo; c0 < hi; c0 += 16) {
        float a[16];
        __syncwarp();
        tmem_ld16(taddr + c0, a);
        if constexpr (PAIR) {
            // lanes 0-15 hold gate, 16-31 up: of each two rows, the lower half takes the first and the upper half the second
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float recv = __shfl_xor_sync(0xffffffffu, upper ? a[2 * j] : a[2 * j + 1], 16);
                y[j] = gated(p, upper ? recv : a[2 * j], upper ? a[2 * j + 1] : recv);
            }
            T* r = upper ? o + p.ldo : o;
            const int left = hi - c0 - (upper ? 1 : 0);
            if (live)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (2 * j < left) st_f(r + (size_t)(2 * j) * p.ldo, y[j]);
        } else if (live) {
            if (p.act == ACT_SILU) {                     // (no activation)
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (c0 + j < hi) st_f(o + (size_t)j * p.ldo, a[j] + bias);
            } else
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (c0 + j < hi) st_f(o + (size_t)j * p.ldo, plain_act(p.act, a[j] + bias));
        }
        o += (size_t)16 * p.ldo;
    }
}

// WIDE: columns [lo, hi) of a finished tile by one warp, its lanes the rows 32 q..
template <bool PAIR, typename T>
__device__ __forceinline__ void store_columns(const Args& p, T* out, const Tile& t, uint32_t taddr, int q, int lane, int lo, int hi) {
    constexpr int OUT = PAIR ? 16 : 32;                  // outputs of 32 columns
    const bool live = 32 * q + lane < t.rows;
    T* o = out + (size_t)(t.row0 + 32 * q + lane) * p.ldo;
    for (int c0 = lo; c0 < hi; c0 += 32) {
        const int n = PAIR ? t.ft * 128 + c0 / 2 : t.ft * 256 + c0;
        if (n >= p.N) break;
        float a[32];
        __syncwarp();
        tmem_ld32(taddr + c0, a);
        if constexpr (PAIR) {
#pragma unroll
            for (int j = 0; j < 16; j++) a[j] = gated(p, a[j], a[j + 16]);
        } else {
            if (p.bias)
#pragma unroll
                for (int j = 0; j < OUT; j++) a[j] += n + j < p.N ? __ldg(p.bias + n + j) : 0.f;
            if (p.act != ACT_SILU)                       // (no activation)
#pragma unroll
                for (int j = 0; j < OUT; j++) a[j] = plain_act(p.act, a[j]);
        }
        if (!live) continue;
        if (p.vec && n + OUT <= p.N) {
            constexpr int UNIT = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < OUT; j += UNIT) {
                uint4 u;
                if constexpr (sizeof(T) == 2) {
                    __nv_bfloat162 h[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(a[j + 2 * i], a[j + 2 * i + 1]);
                    u = *reinterpret_cast<const uint4*>(h);
                } else
                    u = make_uint4(__float_as_uint(a[j]), __float_as_uint(a[j + 1]), __float_as_uint(a[j + 2]), __float_as_uint(a[j + 3]));
                *reinterpret_cast<uint4*>(o + n + j) = u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < OUT; j++)
                if (n + j < p.N) st_f(o + n + j, a[j]);
        }
    }
}

template <int GROUP, bool PAIR, bool WIDE>
__global__ void __launch_bounds__(Form<WIDE>::THREADS, 1)
gemm_q4_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ Args p) {
    using F = Form<WIDE>;
    constexpr int TEAMS = F::TEAMS, PREFETCH = F::PREFETCH, DEQUANT_WARPS = F::DEQUANT_WARPS, EPI_WARPS = F::EPI_WARPS, WARPS = F::WARPS, THREADS = F::THREADS;
    extern __shared__ uint8_t smem_raw[];
    __shared__ volatile int s_abort;
    __shared__ uint32_t s_tmem;
    __shared__ int s_offs[MAX_GROUPS + 1], s_prefix[MAX_GROUPS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ __align__(8) unsigned long long s_bars[2 * STAGES_MAX + 2 * NBUF + 1];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, bars = smem_u32(s_bars);
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (STAGES_MAX + s); };
    auto acc_full = [&](int b) { return bars + 8u * (2 * STAGES_MAX + b); };
    auto acc_empty = [&](int b) { return bars + 8u * (2 * STAGES_MAX + NBUF + b); };
    const uint32_t drained = bars + 8u * (2 * STAGES_MAX + 2 * NBUF);
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < p.stages; s++) mbar_init(full(s), 1 + F::TEAM), mbar_init(empty(s), 1);      // the copies of x, and the warps of values
        for (int b = 0; b < NBUF; b++) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), EPI_WARPS);
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == WARPS - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    int m_tiles = (p.M + p.bn - 1) / p.bn;
    if (p.offsets) {
        pdl_sync();
        for (int i = threadIdx.x; i <= p.G; i += THREADS) s_offs[i] = min(p.M, max(0, p.offsets[i]));
        __syncthreads();
        if (warp == 0) {                                 // row tiles of the groups before each
            int run = 0;
            for (int g0 = 0; g0 < p.G; g0 += 32) {
                const int g = g0 + lane, n = g < p.G ? max(0, s_offs[g + 1] - s_offs[g] + p.bn - 1) / p.bn : 0;
                int upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (g < p.G) s_prefix[g] = run + upto - n;
                run = min(run + __shfl_sync(0xffffffffu, upto, 31), 1 << 29);
            }
            // (offsets that do not ascend may give more than the host checked: nothing is done then)
            if (lane == 0) s_prefix[p.G] = run <= min(p.M, p.G) + p.M / p.bn ? run : 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    if (p.offsets) m_tiles = s_prefix[p.G];
    const int items = m_tiles * p.n_tiles, rank = !WIDE && p.splits > 1 ? (int)cluster_ctarank() : 0;
    const int kb0 = rank * p.kb_per_split, kbs = min(p.w.blocks, kb0 + p.kb_per_split) - kb0;
    const int mine = (int)blockIdx.x < items ? (items - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;      // tiles of this CTA
    const int total = mine * kbs;

    if (warp < DEQUANT_WARPS) {
        // ---- codes to values: block `it` of the CTA's sequence by the warps of team it % TEAMS -----------------------------------------
        if (!p.offsets && !p.early) pdl_wait();
        const int q = warp % F::TEAM, r = lane >> 2, half = PAIR ? p.w.strips / 2 : p.w.strips;
        uint4 code[PREFETCH][2];
        q4::Scales<GROUP> sc[PREFETCH][2];
        int li = 0, kb = warp / F::TEAM;                 // the next block to ask for: tile of this CTA, block of its k
        const uint4* nc[2];
        const uint32_t* ns[2];
        auto aim = [&]() {
            while (kb >= kbs && li < mine) kb -= kbs, li++;
            if (li >= mine) return;
            const Tile t = tile_of(blockIdx.x + li * gridDim.x, m_tiles, p, s_prefix, s_offs);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int strip = PAIR ? t.ft * F::TEAM + q : t.ft * F::TEAM * 2 + 2 * q + i;
                // (strips beyond the last: any values will do, their features are not stored)
                const size_t s = (size_t)t.g * p.w.strips + min(strip, half - 1) + (PAIR && i ? half : 0);
                nc[i] = p.w.codes + (s * p.w.blocks + kb0 + kb) * 32 + lane;
                ns[i] = p.w.scales + s * p.w.qgroups * 8;
            }
        };
        aim();
        auto load = [&](int d) {                         // that block into place d
            if (li < mine) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    code[d][i] = __ldg(nc[i]);
                    sc[d][i].load(ns[i], kb0 + kb, p.w.qgroups, r);
                    nc[i] += TEAMS * 32;
                }
                kb += TEAMS;
                if (kb >= kbs) aim();
            }
        };
#pragma unroll
        for (int d = 0; d < PREFETCH; d++) load(d);
        bool ok = p.test_fault != 3;
        // this lane's place in the tile of values: rows 32 q + r (and 8, 16, 24 further on), the piece of four k at 4 t of the first 16 k (odd rows: the third)
        const bool odd = r & 1;
        const uint32_t place = (uint32_t)((32 * q + r) * 128 + ((((lane & 3) >> 1) ^ r ^ (odd ? 4 : 0)) << 4) + (lane & 1) * 8);
        int s = warp / F::TEAM % p.stages;
        uint32_t parity = 1;
        for (int it0 = warp / F::TEAM; it0 < total && ok; it0 += TEAMS * PREFETCH) {
#pragma unroll
            for (int d = 0; d < PREFETCH; d++) {
                const int it = it0 + TEAMS * d;
                if (it >= total || !ok) break;
                ok = __all_sync(0xffffffffu, mbar_wait(empty(s), parity, &s_abort, p, 0x56));
                if (!ok) break;
                const uint32_t to = base + s * p.stage_bytes + place;
#pragma unroll
                for (int i = 0; i < 2; i++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {        // odd rows take the 16 k in the order 2, 3, 0, 1
                        uint32_t a[4];
                        q4::unpack(odd ? q4::word(code[d][i], j ^ 2) : q4::word(code[d][i], j), p.bits, a);
                        const uint32_t s2 = GROUP == 32 ? (odd != (j >= 2) ? sc[d][i].s[q4::Scales<GROUP>::N - 1] : sc[d][i].s[0]) : sc[d][i].s[0];
                        q4::scale(a, s2);
                        q4::sts8((to ^ (j << 5)) + i * 2048, make_uint2(a[0], a[2]));
                        q4::sts8((to ^ (j << 5)) + i * 2048 + 1024, make_uint2(a[1], a[3]));
                    }
                }
                load(d);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the tensor core reads what was written
                __syncwarp();
                if (lane == 0) mbar_arrive(full(s));
                s += TEAMS;
                if (s >= p.stages) s -= p.stages, parity ^= 1;
            }
        }
        if (!ok && p.test_fault != 3) s_abort = 1;
    } else if (warp < DEQUANT_WARPS + EPI_WARPS) {
        // ---- epilogue -------------------------------------------------------------------------------------------------------------------
        if (WIDE || p.splits == 1) {
            const int q = warp & 3, h = (warp - DEQUANT_WARPS) >> 2;
            bool ok = true;
            for (int li = 0; li < mine && ok; li++) {
                const Tile t = tile_of(blockIdx.x + li * gridDim.x, m_tiles, p, s_prefix, s_offs);
                const int b = li % NBUF;
                ok = mbar_wait(acc_full(b), (li / NBUF) & 1, &s_abort, p, 0x55);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem + b * BN + ((uint32_t)(q * 32) << 16);
                if constexpr (WIDE) {
                    constexpr int PART = 4 * F::FEATURES / EPI_WARPS;
                    if (32 * q < t.rows) {
                        if (p.out_bf16)
                            store_columns<PAIR>(p, (__nv_bfloat16*)p.out, t, taddr, q, lane, h * PART, h * PART + PART);
                        else
                            store_columns<PAIR>(p, (float*)p.out, t, taddr, q, lane, h * PART, h * PART + PART);
                    }
                } else {
                    const int part = ((t.rows + 31) / 32) * 16, lo = min(t.rows, h * part), hi = min(t.rows, lo + part);
                    if (p.out_bf16)
                        store_part<PAIR>(p, (__nv_bfloat16*)p.out, t, taddr, q, lane, lo, hi);
                    else
                        store_part<PAIR>(p, (float*)p.out, t, taddr, q, lane, lo, hi);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(b));
            }
            if (!ok) s_abort = 1;
        }
    } else if (warp == WARPS - 2) {
        // ---- rows of x -------------------------------------------------------------------------------------------------------------------
        if (lane == 0) {
            if (!p.offsets) pdl_sync();
            int it = 0, s = 0;
            uint32_t parity = 1;
            bool ok = p.test_fault != 1;
            for (int li = 0; li < mine && ok; li++) {
                const Tile t = tile_of(blockIdx.x + li * gridDim.x, m_tiles, p, s_prefix, s_offs);
                const int boxes = (t.rows + BOX - 1) / BOX;
                for (int kb = 0; kb < kbs; kb++, it++) {
                    ok = mbar_wait(empty(s), parity, &s_abort, p, 0x51);
                    if (!ok) break;
                    mbar_expect_tx(full(s), boxes * BOX_BYTES);
                    for (int c = 0; c < boxes; c++) tma_load_2d(base + s * p.stage_bytes + F::W_BYTES + c * BOX_BYTES, &tmX, (kb0 + kb) * BK, t.row0 + c * BOX, full(s));
                    if (++s == p.stages) s = 0, parity ^= 1;
                }
            }
            if (!ok && p.test_fault != 1) s_abort = 1;
            // Copies in flight must land before the block leaves.  Where the values do not come, this waits for as long as any wait may: they have landed then.
            for (int i = max(0, it - p.stages); i < it; i++)
                if (!mbar_wait(full(i % p.stages), (i / p.stages) & 1, nullptr, p, 0x52)) break;
        }
    } else {
        // ---- products --------------------------------------------------------------------------------------------------------------------
        if (lane == 0) {
            int s = 0;
            uint32_t parity = 0;
            bool ok = p.test_fault != 2;
            for (int li = 0; li < mine && ok; li++) {
                const Tile t = tile_of(blockIdx.x + li * gridDim.x, m_tiles, p, s_prefix, s_offs);
                const uint32_t idesc = instr_desc(WIDE ? 256 : (t.rows + 15) & ~15);
                const int b = li % NBUF;
                ok = mbar_wait(acc_empty(b), ((li / NBUF) & 1) ^ 1, &s_abort, p, 0x53);
                if (!ok) break;
                for (int kb = 0; kb < kbs; kb++) {
                    ok = mbar_wait(full(s), parity, &s_abort, p, 0x54);
                    if (!ok) break;
                    tc_fence_after();
                    // (WIDE: rows of x beyond the tile's are whatever lies there: lanes that nobody stores)
                    const uint32_t values = base + s * p.stage_bytes, rows = values + F::W_BYTES;
#pragma unroll
                    for (int k4 = 0; k4 < BK / 16; k4++)
                        umma(tmem + b * BN, smem_desc((WIDE ? rows : values) + k4 * 32), smem_desc((WIDE ? values : rows) + k4 * 32), idesc, kb > 0 || k4 > 0);
                    umma_commit(empty(s));
                    if (++s == p.stages) s = 0, parity ^= 1;
                }
                if (ok) umma_commit(acc_full(b));
            }
            if (!ok && p.test_fault != 2) s_abort = 1;
            umma_commit(drained);                        // tensor memory is given back only behind the last product
            mbar_wait(drained, 0, nullptr, p, 0x58);
        }
        __syncwarp();
    }
    if (!WIDE && p.splits > 1) {
        // ---- a tile's k splits: rows [r cpo, (r + 1) cpo) of the tile belong to rank r ------------------------------------------------------
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        const Tile t = tile_of(blockIdx.x, m_tiles, p, s_prefix, s_offs);
        const int S = p.splits, cpo = (t.rows + S - 1) / S;
        if (warp >= DEQUANT_WARPS && warp < DEQUANT_WARPS + EPI_WARPS) {      // the stages are free: the partial tile, [row][features]
            const int q = warp & 3, h = (warp - DEQUANT_WARPS) >> 2;
            const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
            const int part = ((t.rows + 31) / 32) * 16;
            const int lo = min(t.rows, h * part), hi = min(t.rows, lo + part);
            for (int c0 = lo; c0 < hi; c0 += 16) {
                float a[16];
                __syncwarp();
                tmem_ld16(taddr + c0, a);
                const uint32_t to = base + (uint32_t)(c0 * 128 + q * 32 + lane) * 4u;
#pragma unroll
                for (int j = 0; j < 16; j++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + j * 128 * 4), "f"(a[j]) : "memory");
            }
        }
        __syncwarp();
        cluster_sync_all();
        // four features a thread: one 16-byte read of every peer's memory
        const int first = rank * cpo, cols = min(cpo, t.rows - first), per = PAIR ? 16 : 32;
        for (int i = threadIdx.x; i < cols * per; i += THREADS) {
            const int c = i / per, f = (i - c * per) * 4, n = t.ft * per * 4 + f;
            const uint32_t at = base + (uint32_t)((first + c) * 128 + (PAIR ? (f >> 4) * 32 + (f & 15) : f)) * 4u;
            float4 v[MAX_CLUSTER], w[PAIR ? MAX_CLUSTER : 1];
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; s++)
                if (s < S) {
                    const uint32_t peer = mapa_cluster(at, s);
                    v[s] = ld_cluster_f32x4(peer);
                    if constexpr (PAIR) w[s] = ld_cluster_f32x4(peer + 64);
                }
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; s++)
                if (s < S) {
                    x.x += v[s].x, x.y += v[s].y, x.z += v[s].z, x.w += v[s].w;
                    if constexpr (PAIR) y.x += w[s].x, y.y += w[s].y, y.z += w[s].z, y.w += w[s].w;
                }
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < p.N) put(p, t.row0 + first + c, n + e, PAIR ? gated(p, xs[e], ys[e]) : plain_act(p.act, p.bias ? xs[e] + p.bias[n + e] : xs[e]));
        }
        cluster_sync_all();                              // nobody leaves while its memory is read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == WARPS - 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &st) != cudaSuccess || st != cudaDriverEntryPointSuccess) return (EncodeTiledFn) nullptr;
        return (EncodeTiledFn)f;
    }();
    return fn;
}

uint32_t g_wait_limit = WAIT_LIMIT_US;
int g_test_fault = 0;

template <int GROUP, bool PAIR, bool WIDE>
int launch(const CUtensorMap& map, const Args& p, unsigned ctas, cudaStream_t stream) {
    static q4::SmemLimit limit;
    if (const int e = limit.lift((const void*)gemm_q4_tc_kernel<GROUP, PAIR, WIDE>)) return e;
    return launch_pdl_cluster(gemm_q4_tc_kernel<GROUP, PAIR, WIDE>, dim3(ctas, 1, p.splits), dim3(Form<WIDE>::THREADS), (size_t)(p.stages * p.stage_bytes + 1024), stream, p.splits, map, p);
}

}  // namespace

// The same product as moe_gemm_q4 by the kernel above.  Returns -1, with nothing launched, for what it does not take: K or a row pitch of x that is no
// multiple of 8, an unaligned x, more than 1,024 groups.  splits: CTAs of a cluster that share a dense tile's k, 1 to 4.
MOE_API int moe_gemm_q4_tc(const void* x, int ldx, int M, const void* codes, const void* scales, int G, int N, int K, int group, int pair, void* out,
                           int out_bf16, int ldo, const float* bias, const int* offsets, int act, float act_param, int splits, int early, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !codes || !scales || !out || K <= 0 || G <= 0 || (G > 1 && !offsets) || (pair && N % 2)) return (int)cudaErrorInvalidValue;
    if (K % 8 || ldx % 8 || ((uintptr_t)x & 15) || G > MAX_GROUPS || !encode_fn()) return -1;
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)M}, strides[1] = {(cuuint64_t)ldx * 2};
    const cuuint32_t box[2] = {BK, 64}, estr[2] = {1, 1};
    if (encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return -1;
    Args p = {};
    p.w.codes = (const uint4*)codes, p.w.scales = (const uint32_t*)scales, p.w.N = N, p.w.K = K;
    p.N = pair ? N / 2 : N;
    p.w.strips = (p.N + 15) / 16 * (pair ? 2 : 1), p.w.blocks = (K + 63) / 64, p.w.qgroups = (K + group - 1) / group;
    p.out = out, p.out_bf16 = out_bf16, p.ldo = ldo, p.bias = bias, p.offsets = offsets, p.G = G, p.M = M;
    p.act = act, p.act_param = act_param, p.early = early, p.status = status, p.wait_limit = g_wait_limit, p.test_fault = g_test_fault, p.bits = q4::bits();
    // Groups that mostly fit 128 rows take the wide tile.  (us, narrow / wide: 60 experts of a pair 2,816 x 2,048 at 34 rows an expert 126 / 101, at 100 137 / 109,
    // at 136, where most have a second tile, 149 / 177; of 2,048 x 1,408 69 / 52, 73 / 61, 76 / 86.  A dense product of 64 rows of 6,144 x 2,048 in the better
    // number of splits 11.1 / 10.8, of 113 rows 12.1 / 12.4: the narrow one throughout.)
    const int mean = (M + G - 1) / G;
    const bool wide = offsets && mean * 5 / 4 <= 128;
    const int features = (wide ? 256 : 128) / (pair ? 2 : 1);
    p.n_tiles = (p.N + features - 1) / features;
    p.vec = ((uintptr_t)out & 15) == 0 && (long long)ldo * (out_bf16 ? 2 : 4) % 16 == 0;
    // Rows of a tile: as few tiles as 256 rows allow, of equal height.  Groups: what holds a group of half as many rows again as the mean (a smaller tile
    // leaves room for more stages, and the copies' latency counts).
    const int mt = (M + BN - 1) / BN;
    p.bn = wide ? 128 : offsets ? min(BN, (mean * 3 / 2 + BOX - 1) / BOX * BOX) : ((M + mt - 1) / mt + 15) / 16 * 16;
    p.stage_bytes = (wide ? Form<true>::W_BYTES : Form<false>::W_BYTES) + (p.bn + BOX - 1) / BOX * BOX_BYTES;
    p.stages = min(STAGES_MAX, ROOM / p.stage_bytes);
    const int sms = q4::sm_count();
    const long long tiles = (offsets ? (long long)(M < G ? M : G) + M / p.bn : (long long)((M + p.bn - 1) / p.bn)) * p.n_tiles;
    if (tiles > 0x3fffffff) return -1;
    if (offsets || splits < 1) splits = 1;
    if (splits > MAX_CLUSTER) splits = MAX_CLUSTER;
    if (splits > p.w.blocks) splits = p.w.blocks;
    p.kb_per_split = (p.w.blocks + splits - 1) / splits;
    p.splits = (p.w.blocks + p.kb_per_split - 1) / p.kb_per_split;
    const unsigned ctas = p.splits > 1 ? (unsigned)tiles : (unsigned)(tiles < sms ? tiles : sms);
#define GO(GR)                                                                                                  \
    (wide ? (pair ? launch<GR, true, true>(map, p, ctas, stream) : launch<GR, false, true>(map, p, ctas, stream)) \
          : (pair ? launch<GR, true, false>(map, p, ctas, stream) : launch<GR, false, false>(map, p, ctas, stream)))
    switch (group) {
        case 32: return GO(32);
        case 64: return GO(64);
        case 128: return GO(128);
    }
#undef GO
    return (int)cudaErrorInvalidValue;
}

// For the test of the bounded waits only: ``fault`` 1: nothing of x is loaded, 2: no product is issued, 3: no values are formed, so that the other
// roles' waits run out after ``wait_limit`` microseconds (0: the normal limit).  (0, 0) restores the normal behaviour.
MOE_API void moe_q4_set_wait_test(int fault, unsigned wait_limit) {
    g_test_fault = fault >= 1 && fault <= 3 ? fault : 0;
    g_wait_limit = wait_limit ? wait_limit : WAIT_LIMIT_US;
    q4::few_rows_wait_test(g_test_fault, g_wait_limit);
}
