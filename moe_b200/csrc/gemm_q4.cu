// Products of few rows over weights held in 4 bits (the format: quant4.cuh), and a layer of routed experts of few tokens.
//
//   y[m, n] = sum_k x[m, k] q[n, k] s[n, k / group] (+ b[n]), or act(gate) * up of a pair's two rows.
//
// What should bound them is the stream of codes, 0.53 bytes an element; for one row of a long matrix it is the issue slots and the logic unit (without forming
// fragments 27 us of 37): 6.5 TB/s are 46 elements a cycle and SM, and turning eight codes into fragments takes 11 instructions a lane.  So the weights are the A operand of m16n8k16 products
// straight from the registers that they come in (a shift, a mask and a subtraction a pair of elements), a product takes eight rows of x for the
// price of one, and the scale is applied to the sums of a group's k (up to four products from zero, then one multiply-add an output), which also
// keeps the sums in plain 32-bit additions but for those 64.  The warps that share a strip's k add their sums up through shared memory in the order of the warps.
//
//   gemm_q4_direct_kernel    few strips: a block of eight warps a strip, codes and rows straight to registers, all asked for at once.  8 rows of
//                            6,144 x 2,048 3.5 us (with a bias 3.6), 1 row of 2,048 x 2,048 2.4
//   gemm_q4_stream_kernel    many: one block an SM, its codes by bulk copies into stages, the rows' fragments in shared memory.  1 row of
//                            151,936 x 2,048 37 us (4.5 TB/s; ALU 58 %, issue slots 64 %), 16 rows of a pair 40,960 x 3,584 26 us (2.9 TB/s: two rounds of units
//                            with 86 % of the teams' places used, two stages a team at this K; without fragments and products 20.7), 256 rows of 60 experts 2,048 x 1,408 30 us (3.1 TB/s)
//   experts_down_kernel      the second half of a layer of experts.  A layer of 60 experts of 1,408 and a shared one of 5,632, width 2,048: 1 token
//                            18.2 us, 8 tokens 44.6
#include "quant4.cuh"

namespace {

using q4::Weight;
using q4::lds16;
using q4::lds4;
using q4::smem_u32;
using q4::sts8;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four neighbouring k of a row, zeros beyond K or where there is no row.
__device__ __forceinline__ uint2 row4(const __nv_bfloat16* row, int k, int K, int vec) {
    if (!row || k >= K) return make_uint2(0u, 0u);
    if (vec) return *reinterpret_cast<const uint2*>(row + k);
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; i++) e[i] = k + i < K ? (uint32_t)__bfloat16_as_ushort(row[k + i]) : 0u;
    return make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
}

// acc += 64 k of MT strips against NT tiles of eight rows (x[n][j]: the B registers of 16 k), the group's scale on the sums of its k, or, for more than two
// tiles, on the weights (q s is a bfloat16), which saves the registers of a group's sums.  The strips' products alternate: one waits for itself.
template <int MT, int NT, int GROUP>
__device__ __forceinline__ void block_product(const uint4 (&code)[MT], const uint32_t (&sc)[MT][q4::Scales<GROUP>::N], const uint2 (&x)[NT][4], const q4::Bits& bits,
                                              float (&acc)[MT][NT][4]) {
    constexpr int SETS = q4::Scales<GROUP>::N, WORDS = 4 / SETS;
    if constexpr (NT > 2) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int m = 0; m < MT; m++) {
                uint32_t a[4];
                q4::unpack(q4::word(code[m], j), bits, a);
                q4::scale(a, sc[m][j / WORDS]);
#pragma unroll
                for (int n = 0; n < NT; n++) q4::mma(acc[m][n], a, x[n][j].x, x[n][j].y, acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
            }
        return;
    }
#pragma unroll
    for (int h = 0; h < SETS; h++) {
        float c[MT][NT][4];
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            const int j = h * WORDS + i;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                uint32_t a[4];
                q4::unpack(q4::word(code[m], j), bits, a);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if (i == 0)
                        q4::mma(c[m][n], a, x[n][j].x, x[n][j].y, 0.f, 0.f, 0.f, 0.f);
                    else
                        q4::mma(c[m][n], a, x[n][j].x, x[n][j].y, c[m][n][0], c[m][n][1], c[m][n][2], c[m][n][3]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float lo = q4::scale_lo(sc[m][h]), hi = q4::scale_hi(sc[m][h]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                acc[m][n][0] = fmaf(lo, c[m][n][0], acc[m][n][0]), acc[m][n][1] = fmaf(lo, c[m][n][1], acc[m][n][1]);
                acc[m][n][2] = fmaf(hi, c[m][n][2], acc[m][n][2]), acc[m][n][3] = fmaf(hi, c[m][n][3], acc[m][n][3]);
            }
        }
    }
}

// The sums of a team's warps over one tile of eight rows: red [W][MT][8][17] (features of the strip fastest)
template <int MT>
__device__ __forceinline__ void leave_sums(float* red, int warp, int lane, int m, const float (&acc)[4]) {
    const int r = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; i++) red[((warp * MT + m) * 8 + 2 * t + (i & 1)) * 17 + r + 8 * (i >> 1)] = acc[i];
}
template <int W, int MT>
__device__ __forceinline__ float sum_of(const float* red, int m, int col, int row) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) v += red[((w * MT + m) * 8 + col) * 17 + row];
    return v;
}
template <int THREADS>
__device__ __forceinline__ void team_sync(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}

// the same, and whether every warp says so
template <int THREADS>
__device__ __forceinline__ bool team_sync_and(int id, bool mine) {
    int all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 q, %1, 0;\n\tbar.red.and.pred p, %2, %3, q;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(all) : "r"((int)mine), "r"(id), "n"(THREADS) : "memory");
    return all != 0;
}

// ---- the picked experts of a step of few tokens -------------------------------------------------------------------------------------------
constexpr int EXPERTS_MAX = 1024, FEW = 8, PAIRS_MAX = 128;
struct Picked {
    uint32_t bits[EXPERTS_MAX / 32];
    int before[EXPERTS_MAX / 32 + 1];      // picked experts below each word
    short pick[PAIRS_MAX];                 // the expert of a pair, -1 for none
    short expert[PAIRS_MAX];               // of a slot: the picked experts in order of their numbers
    uint32_t takes[PAIRS_MAX + 1];         // of a slot: the tokens that picked it; behind the last slot: all, for the shared expert
    __device__ __forceinline__ int slot_of(int e) const { return before[e >> 5] + __popc(bits[e >> 5] & ((1u << (e & 31)) - 1)); }
};
// By one warp; the block's other threads read it behind a barrier.
__device__ __forceinline__ void find_picked(const int* idx, int T, int top_k, int E, int* status, Picked& s, int lane) {
    const int pairs = T * top_k;
    s.bits[lane] = 0;
    __syncwarp();
    for (int i = lane; i < pairs; i += 32) {
        int e = idx[i];
        s.takes[i] = 0;
        if (e >= 0 && e < E)
            atomicOr(&s.bits[e >> 5], 1u << (e & 31));
        else {
            if (e != -1 && status) atomicOr(status, ST_BAD_EXPERT);
            e = -1;
        }
        s.pick[i] = (short)e;
    }
    __syncwarp();
    const int n = __popc(s.bits[lane]);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    s.before[lane] = upto - n;
    if (lane == 31) s.before[32] = upto;
    __syncwarp();
    for (int i = lane; i < pairs; i += 32) {
        const int e = s.pick[i];
        if (e < 0) continue;
        const int slot = s.slot_of(e);
        s.expert[slot] = (short)e;
        atomicOr(&s.takes[slot], 1u << (i / top_k));
    }
    if (lane == 0) s.takes[s.before[32]] = (1u << T) - 1;
    __syncwarp();
}

struct Args {
    Weight w, shared;              // shared: EXPERTS, codes null where there is none
    const __nv_bfloat16* x;        // [M, K], pitch ldx; vec: rows of whole 8-byte units
    int ldx, vec, M;
    void* out;
    int out_bf16, ldo, N;          // N: output features (of a pair: of one half)
    const float* bias;
    const int* offsets;
    int G;
    int act;
    float act_param;
    const int* idx;                // EXPERTS: the picks, [M, top_k]
    int top_k, E;
    uint8_t *frag, *sfrag;         // EXPERTS: [slot][frag_blocks] of TERMS_BLOCK bytes, see experts_down_kernel; the shared expert's
    int frag_blocks;
    int early;                     // the weights may be read before what is in front of this launch has ended
    q4::Bits bits;
    q4::Waits waits;
};

__device__ __forceinline__ void put(const Args& p, int row, int n, float y) {
    const size_t o = (size_t)row * p.ldo + n;
    if (p.out_bf16)
        ((__nv_bfloat16*)p.out)[o] = __float2bfloat16_rn(y);
    else
        ((float*)p.out)[o] = y;
}

// ---- few strips -----------------------------------------------------------------------------------------------------------------------------
// Grid: strips of the output (of a pair: of one half).  Warp w takes blocks w, w + 8, ... of 64 k, DEPTH of them in flight; the codes are asked for
// before the wait on the predecessor, the rows behind it and one block ahead.  Three blocks an SM count for more than anything that their registers
// could hold.  (us of one set of runs, two / three: 8 rows of 6,144 x 2,048, with all four blocks' rows ahead in the first, 6.3 / 3.6, of a pair 11,264 x 2,048 6.7 / 4.8,
// of 2,048 x 5,632 4.8 / 5.6; 16 rows 8.9 / 6.5, 10.6 / 8.7, 9.0 / 8.8; 24 rows 8.9 / 8.4, 14.7 / 12.5, 12.5 / 12.0.)
template <int MT, int NT, int GROUP>
__global__ void __launch_bounds__(256, 3)
gemm_q4_direct_kernel(const __grid_constant__ Args p) {
    constexpr int W = 8, DEPTH = MT == 2 && NT > 1 ? 2 : 4, NS = q4::Scales<GROUP>::N;
    __shared__ float red[W * MT * 8 * 17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, strip = blockIdx.x, blocks = p.w.blocks;
    const uint4* codes[MT];
    const uint32_t* scales[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const size_t s = strip + m * (p.w.strips / 2);
        codes[m] = p.w.codes + s * blocks * 32 + lane;
        scales[m] = p.w.scales + s * p.w.qgroups * 8;
    }
    bool waited = !p.early;
    if (waited) pdl_sync();
    for (int row0 = 0; row0 < p.M; row0 += 8 * NT) {
        uint4 code[DEPTH][MT];
        uint32_t sc[DEPTH][MT][NS];
        uint2 x[NT][4];                                  // one block ahead
        const __nv_bfloat16* xr[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) xr[n] = row0 + 8 * n + r < p.M ? p.x + (size_t)(row0 + 8 * n + r) * p.ldx : nullptr;
        auto ask = [&](int d, int b) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(code[d][m].x), "=r"(code[d][m].y), "=r"(code[d][m].z), "=r"(code[d][m].w)
                             : "l"(codes[m] + (size_t)b * 32));
                q4::Scales<GROUP> s;
                s.load(scales[m], b, p.w.qgroups, r);
#pragma unroll
                for (int i = 0; i < NS; i++) sc[d][m][i] = s.s[i];
            }
        };
        auto ask_rows = [&](int b) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) x[n][j] = row4(xr[n], b * 64 + 16 * j + 4 * t, p.w.K, p.vec);
        };
        float acc[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (warp + d * W < blocks) ask(d, warp + d * W);
        if (!waited) pdl_sync();
        waited = true;
        if (warp < blocks) ask_rows(warp);
        for (int b0 = warp; b0 < blocks; b0 += DEPTH * W) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                const int b = b0 + d * W;
                if (b >= blocks) break;
                block_product<MT, NT, GROUP>(code[d], sc[d], x, p.bits, acc);
                if (b + W < blocks) ask_rows(b + W);
                if (b + DEPTH * W < blocks) ask(d, b + DEPTH * W);
            }
        }
#pragma unroll
        for (int n8 = 0; n8 < NT; n8++) {
#pragma unroll
            for (int m = 0; m < MT; m++) leave_sums<MT>(red, warp, lane, m, acc[m][n8]);
            __syncthreads();
            const int i = threadIdx.x, col = i >> 4, f = i & 15, n = strip * 16 + f, row = row0 + 8 * n8 + col;
            if (i < 128 && n < p.N && row < p.M) {
                float y = sum_of<W, MT>(red, 0, col, f);
                y = MT == 2 ? glu_mul(p.act, p.act_param, y, sum_of<W, MT>(red, MT - 1, col, f)) : plain_act(p.act, p.bias ? y + p.bias[n] : y);
                put(p, row, n, y);
            }
            __syncthreads();
        }
    }
}

// ---- many strips ----------------------------------------------------------------------------------------------------------------------------
// DENSE   one weight, up to 8 NT rows, NT 1 to 3
// GROUPED rows [offsets[g], offsets[g + 1]) meet weight g, 8 NT at a time
// EXPERTS the gate and up rows of a layer of routed experts: the eight rows of a unit are the step's tokens whatever the expert, so
//         that nothing is gathered; the shared expert's strips come first.  What comes out lies as the B fragments of the next
//         product, as three bfloat16 terms that together are the 32-bit number.
//
// A unit is two strips (a pair's gate and up strip, or neighbours) and up to 8 NT rows.  A block takes a run of neighbouring units; its five teams of
// four warps take them in turn, and the warps of a team every fourth block of 64 k.  One more warp a team has its codes copied (cp.async.bulk) into
// stages of KC blocks, across the borders of units.  The fragments of the rows lie in shared memory for all teams; where the
// rows change (GROUPED), all teams meet.
enum { DENSE = 0, GROUPED = 1, EXPERTS = 2 };
constexpr int TERMS_BLOCK = 3072;      // EXPERTS: bytes of 64 k of eight rows in three terms, see experts_down_kernel
constexpr int GROUPS_MAX = 1024, TEAM_W = 4, TEAMS = 5, KC = 8, STREAM_THREADS = TEAMS * (TEAM_W + 1) * 32, STAGES_MAX = 8;

template <int NT, int GROUP>
struct Stream {
    static constexpr int SCALE_BLOCK = GROUP == 32 ? 64 : GROUP == 64 ? 32 : 16;      // bytes a block of 64 k (128: a pair of blocks has 32)
    static constexpr int CODES = KC * 512, SCALES = KC * SCALE_BLOCK, STAGE = 2 * (CODES + SCALES);
    static constexpr int RED_BUFFERS = NT == 1 ? 2 : 1, RED_FLOATS = TEAM_W * 2 * 8 * 17;      // of a team
    static constexpr int RED = TEAMS * RED_BUFFERS * RED_FLOATS * 4;
    static int bytes(int blocks, int stages) { return TEAMS * stages * STAGE + RED + blocks * NT * 1024; }
};

struct Unit {
    int strip, g, slot;            // first strip (of the half); group; EXPERTS: slot, -1: the shared expert
};

template <int MODE, int NT, int GROUP, bool PAIR>
__global__ void __launch_bounds__(STREAM_THREADS, 1)
gemm_q4_stream_kernel(const __grid_constant__ Args p, const int stages) {
    using S = Stream<NT, GROUP>;
    constexpr int UM = PAIR ? 1 : 2;                      // strips of the output a unit
    extern __shared__ __align__(128) uint8_t smem[];     // the teams' stages, the teams' sums, the rows' fragments [blocks][NT][2][32] x 16 bytes
    __shared__ int s_first[MODE == GROUPED ? GROUPS_MAX + 1 : 1], s_off[MODE == GROUPED ? GROUPS_MAX + 1 : 1];
    __shared__ Picked picked;
    __shared__ __align__(8) unsigned long long s_bars[TEAMS][2][STAGES_MAX], s_ready;
    __shared__ volatile int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = p.w.blocks, half = PAIR ? p.w.strips / 2 : p.w.strips, per = (half + UM - 1) / UM;      // units of a weight and row chunk
    if (threadIdx.x < TEAMS * stages) {
        const int q = threadIdx.x / stages, s = threadIdx.x % stages;
        q4::mbar_init(smem_u32(&s_bars[q][0][s]), 1), q4::mbar_init(smem_u32(&s_bars[q][1][s]), TEAM_W);
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        q4::mbar_init(smem_u32(&s_ready), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // This block's units [u0, u1).  EXPERTS: its part of the shared expert's strips, which is known (and copied) before the picks are, [0, n1), and then its part
    // of the picked experts' from number ea on, [n1, u1).
    auto part = [&](int units, int i) { return (int)((long long)units * i / gridDim.x); };
    const int shared_units = MODE == EXPERTS && p.shared.codes ? p.shared.strips / 2 : 0, sa = part(shared_units, blockIdx.x), n1 = part(shared_units, blockIdx.x + 1) - sa;
    int u0 = 0, u1 = n1, ea = 0;
    // (with a unit a block or more of the picked experts, both parts together are as even as one part would be: a block whose first part was rounded up takes
    // less in the second)
    auto know_picks = [&]() {
        const int units = picked.before[32] * per;
        auto first = [&](int i) {
            const long long over = units >= (int)gridDim.x ? (long long)shared_units * i % gridDim.x : 0;
            return (int)(((long long)units * i + over) / gridDim.x);
        };
        ea = first(blockIdx.x), u1 = n1 + first(blockIdx.x + 1) - ea;
    };
    if (MODE != EXPERTS) {
        int units = per;
        if (MODE == GROUPED) {
            pdl_sync();
            for (int i = threadIdx.x; i <= p.G; i += STREAM_THREADS) s_off[i] = min(p.M, max(0, p.offsets[i]));
            __syncthreads();
            if (warp == 0) {                             // row chunks of the groups before each
                int run = 0;
                for (int g0 = 0; g0 < p.G; g0 += 32) {
                    const int g = g0 + lane, n = g < p.G ? max(0, s_off[g + 1] - s_off[g] + 8 * NT - 1) / (8 * NT) : 0;
                    int upto = n;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += v;
                    }
                    if (g < p.G) s_first[g] = run + upto - n;
                    run = min(run + __shfl_sync(0xffffffffu, upto, 31), 1 << 29);
                }
                // (offsets that do not ascend may give more than the launch was sized for: nothing is done then)
                if (lane == 0) s_first[p.G] = run <= min(p.M, p.G) + p.M / (8 * NT) ? run : 0;
            }
            __syncthreads();
            units = s_first[p.G] * per;
        }
        u0 = part(units, blockIdx.x), u1 = part(units, blockIdx.x + 1);
    }
    __syncthreads();
    auto locate = [&](int u) {
        Unit v;
        v.g = 0, v.slot = 0;
        if (MODE == EXPERTS) {
            if (u < n1)
                v.slot = -1, v.strip = sa + u;
            else
                u += ea - n1, v.slot = u / per, v.strip = u - v.slot * per, v.g = picked.expert[v.slot];
        } else {
            const int c = u / per;
            v.strip = (u - c * per) * UM;
            if (MODE == GROUPED) {
                int lo = 0, hi = p.G;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s_first[mid] <= c) lo = mid; else hi = mid;
                }
                v.g = lo;
            }
        }
        return v;
    };
    // the unit TEAMS further on, u
    auto step = [&](Unit& v, int u) {
        v.strip += TEAMS * UM;
        if (v.strip >= half || (MODE == EXPERTS && v.slot < 0)) v = locate(u);
    };
    // A run: units of the same rows.  GROUPED: a chunk's; else all.
    auto run_end = [&](int u) { return MODE == GROUPED ? min(u1, (u / per + 1) * per) : u1; };
    const int unit_stages = (blocks + KC - 1) / KC;

    if (warp >= TEAMS * TEAM_W) {
        // ---- copies of team q ---------------------------------------------------------------------------------------------------------------
        if (lane || p.waits.test_fault == 1) return;
        if (MODE != GROUPED && !p.early) pdl_wait();
        const int q = warp - TEAMS * TEAM_W;
        int u = u0 + q, end = u0 < u1 ? run_end(u0) : u0, s = 0, it = 0;
        bool waits = MODE == EXPERTS;                    // for the picks
        uint32_t parity = 1;
        const uint32_t base = smem_u32(smem) + q * stages * S::STAGE, bars = smem_u32(&s_bars[q][0][0]);
        bool ok = true;
        while (ok) {
            if (MODE == GROUPED)
                while (u >= end && end < u1) u = end + q, end = run_end(end);      // past its run: the team's first unit of the next one
            if (u >= end) {
                if (!waits) break;
                waits = false;
                if (!(ok = q4::mbar_wait(smem_u32(&s_ready), 0, &s_abort, p.waits.limit_us, p.waits.status, 0x63))) break;
                know_picks();
                end = u1;
                continue;
            }
            for (Unit v = locate(u); ok && u < end;) {
                const Weight& w = MODE == EXPERTS && v.slot < 0 ? p.shared : p.w;
                const size_t s0 = (size_t)v.g * w.strips + v.strip, s1 = PAIR ? s0 + w.strips / 2 : v.strip + 1 < half ? s0 + 1 : s0;
                const uint8_t *c0 = (const uint8_t*)(w.codes + s0 * blocks * 32), *c1 = (const uint8_t*)(w.codes + s1 * blocks * 32);
                const uint8_t *q0 = (const uint8_t*)(w.scales + s0 * w.qgroups * 8), *q1 = (const uint8_t*)(w.scales + s1 * w.qgroups * 8);
                int groups = w.qgroups;                  // left
                for (int kb = 0; kb < blocks; kb += KC) {
                    if (it >= stages && !(ok = q4::mbar_wait(bars + 8 * (STAGES_MAX + s), parity, &s_abort, p.waits.limit_us, p.waits.status, 0x61))) break;
                    const int n = min(KC, blocks - kb) * 512, qn = min(groups, S::SCALES / 32) * 32;
                    const uint32_t to = base + s * S::STAGE, full = bars + 8 * s;
                    q4::mbar_expect_tx(full, 2 * (n + qn));
                    q4::bulk_copy(to, c0, n, full);
                    q4::bulk_copy(to + S::CODES, c1, n, full);
                    q4::bulk_copy(to + 2 * S::CODES, q0, qn, full);
                    q4::bulk_copy(to + 2 * S::CODES + S::SCALES, q1, qn, full);
                    c0 += S::CODES, c1 += S::CODES, q0 += S::SCALES, q1 += S::SCALES, groups -= S::SCALES / 32;
                    it++;
                    if (++s == stages) s = 0, parity ^= 1;
                }
                u += TEAMS;
                if (u < end) step(v, u);
            }
        }
        if (!ok) s_abort = 1;
        for (int i = max(0, it - stages); i < it; i++)      // copies in flight must land before the block leaves
            q4::mbar_wait(bars + 8 * (i % stages), (i / stages) & 1, nullptr, p.waits.limit_us, p.waits.status, 0x62);
        return;
    }

    // ---- products ---------------------------------------------------------------------------------------------------------------------------
    const int team = warp / TEAM_W, tw = warp % TEAM_W, r = lane >> 2;
    const uint32_t base = smem_u32(smem) + team * stages * S::STAGE, xs = smem_u32(smem) + TEAMS * stages * S::STAGE + S::RED;
    float* red = reinterpret_cast<float*>(smem + TEAMS * stages * S::STAGE) + team * S::RED_BUFFERS * S::RED_FLOATS;
    if (MODE != GROUPED) pdl_sync();
    if (MODE == EXPERTS) {
        if (warp == 0) {
            find_picked(p.idx, p.M, p.top_k, p.E, blockIdx.x == 0 ? p.waits.status : nullptr, picked, lane);
            if (lane == 0) q4::mbar_arrive(smem_u32(&s_ready));
        }
        u1 = n1 + 1;                                     // (one run, staged below; how long it is is known behind the barrier there)
    }
    int s = 0, turn = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int first = u0; first < u1; first = run_end(first)) {
        int row0 = 0, rows = p.M;
        if (MODE == GROUPED) {
            const int c = first / per;
            const Unit v = locate(first);
            row0 = s_off[v.g] + (c - s_first[v.g]) * 8 * NT, rows = min(8 * NT, s_off[v.g + 1] - row0);
            if (first > u0) team_sync<TEAMS * TEAM_W * 32>(TEAMS + 1);      // the rows before are done with
        }
        // a thread's four k of all rows are asked for at once
        for (int k4 = threadIdx.x; k4 < blocks * 16; k4 += TEAMS * TEAM_W * 32) {
            uint2 y[8 * NT];
#pragma unroll
            for (int c = 0; c < 8 * NT; c++) y[c] = row4(c < rows ? p.x + (size_t)(row0 + c) * p.ldx : nullptr, k4 * 4, p.w.K, p.vec);
            const int b = k4 >> 4, j = (k4 >> 2) & 3, tt = k4 & 3;
#pragma unroll
            for (int c = 0; c < 8 * NT; c++) sts8(xs + ((b * NT + (c >> 3)) * 2 + (j >> 1)) * 512 + ((c & 7) * 4 + tt) * 16 + (j & 1) * 8, y[c]);
        }
        team_sync<TEAMS * TEAM_W * 32>(TEAMS + 1);
        if (MODE == EXPERTS) know_picks();
        const int end = run_end(first);
        Unit v;
        if (first + team < end) v = locate(first + team);
        for (int u = first + team; u < end && ok; u += TEAMS) {
            if (u > first + team) step(v, u);
            float acc[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
            uint32_t xa = xs + tw * NT * 1024 + lane * 16;
            int left = blocks - tw;                      // blocks from this warp's first on
            for (int st = 0; st < unit_stages; st++) {
                // (a lane may give up where another is let through: the warp goes on, to products that all of it has to reach, or gives up, as a whole)
                ok = __all_sync(0xffffffffu, q4::mbar_wait(smem_u32(&s_bars[team][0][s]), parity, &s_abort, p.waits.limit_us, p.waits.status, 0x64));
                if (!ok) break;
                const uint32_t at = base + s * S::STAGE + tw * 512 + lane * 16, as = base + s * S::STAGE + 2 * S::CODES + r * 4;
#pragma unroll
                for (int i = 0; i < KC / TEAM_W; i++) {
                    if (left > i * TEAM_W) {
                        uint4 code[2];
                        uint32_t sc[2][q4::Scales<GROUP>::N];
                        uint2 x[NT][4];
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            code[m] = lds16(at + m * S::CODES + i * TEAM_W * 512);
                            const uint32_t a = as + m * S::SCALES + (GROUP == 128 ? (tw + i * TEAM_W) / 2 * 32 : (tw + i * TEAM_W) * S::SCALE_BLOCK);
                            sc[m][0] = lds4(a);
                            // (a second group that begins beyond K was not copied; its q are 0)
                            if (GROUP == 32) sc[m][q4::Scales<GROUP>::N - 1] = (st * KC + i * TEAM_W + tw) * 64 + 32 < p.w.K ? lds4(a + 32) : 0u;
                        }
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint4 y = lds16(xa + i * TEAM_W * NT * 1024 + (n * 2 + h) * 512);
                                x[n][2 * h] = make_uint2(y.x, y.y), x[n][2 * h + 1] = make_uint2(y.z, y.w);
                            }
                        block_product<2, NT, GROUP>(code, sc, x, p.bits, acc);
                    }
                }
                left -= KC, xa += KC * NT * 1024;
                __syncwarp();
                if (lane == 0) q4::mbar_arrive(smem_u32(&s_bars[team][1][s]));
                if (++s == stages) s = 0, parity ^= 1;
            }
#pragma unroll
            for (int n8 = 0; n8 < NT; n8++) {
                float* sums = red + (S::RED_BUFFERS == 2 ? turn : 0) * S::RED_FLOATS;
                turn ^= 1;
#pragma unroll
                for (int m = 0; m < 2; m++) leave_sums<2>(sums, tw, lane, m, acc[m][n8]);
                // (two buffers: this one is written again only behind the next one's barrier.  A team gives up as a whole.)
                if (n8 == 0)
                    ok = team_sync_and<TEAM_W * 32>(team + 1, ok);
                else
                    team_sync<TEAM_W * 32>(team + 1);
                if (!ok) s_abort = 1;
#pragma unroll
                for (int o = 0; o < UM * 128; o += TEAM_W * 32) {
                    const int m = o >> 7, i = (o & 127) + tw * 32 + lane, col = i >> 4, f = i & 15, n = (v.strip + m) * 16 + f;
                    if (MODE == EXPERTS) {
                        const bool takes = col < p.M && (v.slot < 0 || ((picked.takes[v.slot] >> col) & 1));
                        float a = 0.f;
                        if (takes) a = glu_mul(ACT_SILU, 0.f, sum_of<TEAM_W, 2>(sums, 0, col, f), sum_of<TEAM_W, 2>(sums, 1, col, f));
                        // a = t[0] + t[1] + t[2]: each cuts eight bits of mantissa off what is left (nothing is rounded, but for what lies below 2^-133)
                        float left = a;
                        uint16_t t[3];
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            const uint32_t cut = __float_as_uint(left) & 0xffff0000u;
                            t[k] = (uint16_t)(cut >> 16), left = isinf(left) ? 0.f : left - __uint_as_float(cut);
                        }
                        const int at = col * 4 + (f >> 2);
                        uint8_t* to = (v.slot < 0 ? p.sfrag : p.frag + (size_t)v.slot * p.frag_blocks * TERMS_BLOCK) + (size_t)(v.strip >> 2) * TERMS_BLOCK;
                        uint16_t *first = reinterpret_cast<uint16_t*>(to + (v.strip & 3) * 512 + at * 16) + (f & 3),
                                 *last = reinterpret_cast<uint16_t*>(to + 2048 + (v.strip & 2) * 256 + at * 16 + (v.strip & 1) * 8) + (f & 3);
                        first[0] = t[0], first[4] = t[1], *last = t[2];
                        // the strips that fill the last block of 64
                        if (v.strip == (v.slot < 0 ? shared_units : half) - 1)
                            for (int z = v.strip + 1; z & 3; z++) {
                                *reinterpret_cast<uint32_t*>(to + (z & 3) * 512 + i * 4) = 0u;
                                if (i < 64) *reinterpret_cast<uint32_t*>(to + 2048 + (z & 2) * 256 + (i >> 1) * 16 + (z & 1) * 8 + (i & 1) * 4) = 0u;
                            }
                        continue;
                    }
                    if (n >= p.N || n8 * 8 + col >= rows) continue;
                    float y = sum_of<TEAM_W, 2>(sums, m, col, f);
                    y = PAIR ? glu_mul(p.act, p.act_param, y, sum_of<TEAM_W, 2>(sums, 1, col, f)) : plain_act(p.act, p.bias ? y + p.bias[n] : y);
                    put(p, row0 + n8 * 8 + col, n, y);
                }
                if (S::RED_BUFFERS == 1) team_sync<TEAM_W * 32>(team + 1);
            }
        }
    }
}

// ---- the down products of a layer of routed experts ---------------------------------------------------------------------------------------
//   out_t = sum_e w_te Wd_e a_te + gate_t Wd_s a_t,  w_te the sum of t's weights for expert e
// Four strips of the output go through ALL picked experts and the shared one, w_te on the sums of each block of 64 k: nothing is left to
// combine.  Tokens that did not pick an expert meet it with the zeros that the first kernel left, and its sums stay out of theirs (a scale may be NaN).  A block of 64 k of the rows is 3 KB: for each
// 16 k a B fragment of 32 lanes x (four k's first terms, their second terms), and behind the four of them the third terms, 8 bytes a lane.  (With two terms, rounded, the
// layer's 32-bit output was 2.4e-6 of its norm off, ten times what its sums leave: 1 token 17.3 us, 8 tokens 41.6, now 18.2, 44.6.  32-bit rows that become three terms
// in registers here: 18.9, 47.0.)  Grid: (fours of strips, 1, S); the S blocks of a unit are
// a cluster and share its blocks of 64 k; the first of them adds their sums up in order.  A warp takes every sixteenth block and copies for itself
// into a ring of its own (cp.async: its pieces of 512 bytes and less are too small for bulk copies, of which an SM issued one in ten to twenty cycles).
constexpr int DOWN_W = 16, DOWN_MT = 4, DOWN_DEPTH = 2, DOWN_THREADS = DOWN_W * 32;
struct DownArgs {
    Weight down, shared;           // shared.codes null: none
    const uint8_t *frag, *sfrag;
    int T, H, E, top_k, S;
    const int* idx;
    const float* wk;
    const float* gate;
    void* out;
    int out_bf16, ldo;
    q4::Bits bits;
};
template <int GROUP>
struct DownRing {
    static constexpr int SCALES = GROUP == 32 ? 64 : 32, X = DOWN_MT * (512 + SCALES), SLOT = X + TERMS_BLOCK, BYTES = DOWN_W * DOWN_DEPTH * SLOT;
    static_assert(DOWN_W * DOWN_MT * 8 * 17 * 4 <= BYTES && DOWN_THREADS == DOWN_MT * 128, "sums");  // they lie over the rings
    static constexpr int PARTS = 7 * DOWN_MT * 128 * 4;             // the other blocks' sums, behind the rings
};

template <int GROUP>
__global__ void __launch_bounds__(DOWN_THREADS, 1)
experts_down_kernel(const __grid_constant__ DownArgs p) {
    using D = DownRing<GROUP>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Picked picked;
    __shared__ float wk[PAIRS_MAX];
    __shared__ __align__(16) float wt[PAIRS_MAX + 1][FEW];      // a slot's weight of each token; the last one's: the shared expert's gate
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, strip0 = blockIdx.x * DOWN_MT, rank = blockIdx.z;
    if (p.S > 1) cluster_arrive();                              // (waited for below: this block's memory may be written to)
    // The picks and the weights were written at least two kernels ago (this one's predecessor let it in behind its own wait): they are read before the
    // wait.
    const int pairs = p.T * p.top_k;
    if (warp == 0)
        find_picked(p.idx, p.T, p.top_k, p.E, nullptr, picked, lane);
    else if (threadIdx.x - 32 < pairs)
        wk[threadIdx.x - 32] = p.wk[threadIdx.x - 32];
    const float gate = threadIdx.x < p.T && p.gate ? p.gate[threadIdx.x] : 1.f;
    __syncthreads();
    const int slots = picked.before[32], nb = p.down.blocks, total = slots * nb + (p.shared.codes ? p.shared.blocks : 0);
    const int lo = (int)((long long)total * rank / p.S), hi = (int)((long long)total * (rank + 1) / p.S);
    const int count = hi - lo > warp ? (hi - lo - warp - 1) / DOWN_W + 1 : 0;      // this warp's blocks

    struct Place {
        int slot, b;
        __device__ __forceinline__ void next(int slots, int nb) {
            b += DOWN_W;
            while (slot < slots && b >= nb) b -= nb, slot++;
        }
    };
    const uint32_t ring = smem_u32(smem) + warp * DOWN_DEPTH * D::SLOT;
    // a lane's piece of the scales: strip lane / (2 NS)
    constexpr int NS = q4::Scales<GROUP>::N;
    int strips[DOWN_MT];
#pragma unroll
    for (int m = 0; m < DOWN_MT; m++) strips[m] = min(strip0 + m, p.down.strips - 1);
    const int scale_strip = min(strip0 + lane / (2 * NS), p.down.strips - 1);
    auto copy_codes = [&](uint32_t to, Place at) {
        const bool own = at.slot < slots;
        const Weight& w = own ? p.down : p.shared;
        const size_t first = (size_t)(own ? picked.expert[at.slot] : 0) * w.strips;
#pragma unroll
        for (int m = 0; m < DOWN_MT; m++) copy16(to + m * 512 + lane * 16, w.codes + ((first + strips[m]) * w.blocks + at.b) * 32 + lane);
        if (lane < DOWN_MT * 2 * NS) {
            const int q = GROUP == 32 ? min(2 * at.b + (lane >> 1) % 2, w.qgroups - 1) : GROUP == 64 ? at.b : at.b >> 1;      // (a group beyond the last: its q are 0)
            copy16(to + DOWN_MT * 512 + lane * 16, reinterpret_cast<const uint4*>(w.scales) + ((first + scale_strip) * w.qgroups + q) * 2 + (lane & 1));
        }
    };
    auto copy_rows = [&](uint32_t to, Place at) {
        const uint8_t* from = (at.slot < slots ? p.frag + (size_t)at.slot * nb * TERMS_BLOCK : p.sfrag) + (size_t)at.b * TERMS_BLOCK + lane * 16;
#pragma unroll
        for (int j = 0; j < 6; j++) copy16(to + D::X + j * 512 + lane * 16, from + j * 512);
    };
    Place now;
    now.slot = min((lo + warp) / nb, slots), now.b = lo + warp - now.slot * nb;
    Place ahead = now;
    for (int i = 0; i < min(count, DOWN_DEPTH - 1); i++, ahead.next(slots, nb)) copy_codes(ring + i * D::SLOT, ahead);
    // the slots' weights (an expert may be picked twice), under the first copies
    for (int i = threadIdx.x; i < slots * FEW; i += DOWN_THREADS) {
        const int e = picked.expert[i >> 3], c = i & 7;
        float v = 0.f;
        if ((picked.takes[i >> 3] >> c) & 1)
            for (int j = c * p.top_k; j < (c + 1) * p.top_k; j++)
                if (picked.pick[j] == e) v += wk[j];
        wt[i >> 3][c] = v;
    }
    if (threadIdx.x < FEW) wt[slots][threadIdx.x] = (int)threadIdx.x < p.T && p.shared.codes ? gate : 0.f;
    pdl_sync();
    ahead = now;
#pragma unroll 1
    for (int i = 0; i < DOWN_DEPTH - 1; i++) {
        if (i < count) copy_rows(ring + i * D::SLOT, ahead), ahead.next(slots, nb);
        copy_commit();                                          // (the codes are part of the first group)
    }
    __syncthreads();

    float acc[DOWN_MT][4] = {};
    uint32_t at = ring, spare = ring + (DOWN_DEPTH - 1) * D::SLOT;
    for (int i = 0; i < count; i++) {
        if (i + DOWN_DEPTH - 1 < count) copy_codes(spare, ahead), copy_rows(spare, ahead), ahead.next(slots, nb);
        copy_commit();
        copy_wait<DOWN_DEPTH - 1>();
        __syncwarp();                                           // (the scales were copied by other lanes)
        float c[DOWN_MT][4], sum[DOWN_MT][4];
        uint4 code[DOWN_MT], third;
#pragma unroll
        for (int m = 0; m < DOWN_MT; m++) code[m] = lds16(at + m * 512 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 two = lds16(at + D::X + j * 512 + lane * 16);
            if (j % 2 == 0) third = lds16(at + D::X + 2048 + j * 256 + lane * 16);
            const uint2 x[3] = {make_uint2(two.x, two.y), make_uint2(two.z, two.w), j % 2 ? make_uint2(third.z, third.w) : make_uint2(third.x, third.y)};
            const bool fresh = GROUP == 32 ? j % 2 == 0 : j == 0, last = GROUP == 32 ? j % 2 == 1 : j == 3;
#pragma unroll
            for (int m = 0; m < DOWN_MT; m++) {
                uint32_t a[4];
                q4::unpack(q4::word(code[m], j), p.bits, a);
#pragma unroll
                for (int i = 0; i < 3; i++) {
                    if (fresh && i == 0)
                        q4::mma(c[m], a, x[i].x, x[i].y, 0.f, 0.f, 0.f, 0.f);
                    else
                        q4::mma(c[m], a, x[i].x, x[i].y, c[m][0], c[m][1], c[m][2], c[m][3]);
                }
            }
            if (last)
#pragma unroll
                for (int m = 0; m < DOWN_MT; m++) {
                    const uint32_t sc = lds4(at + DOWN_MT * 512 + m * D::SCALES + (GROUP == 32 ? j / 2 * 32 : 0) + r * 4);
                    const float l = q4::scale_lo(sc), h = q4::scale_hi(sc);
                    const bool one = GROUP != 32 || j == 1;
                    sum[m][0] = one ? l * c[m][0] : fmaf(l, c[m][0], sum[m][0]), sum[m][1] = one ? l * c[m][1] : fmaf(l, c[m][1], sum[m][1]);
                    sum[m][2] = one ? h * c[m][2] : fmaf(h, c[m][2], sum[m][2]), sum[m][3] = one ? h * c[m][3] : fmaf(h, c[m][3], sum[m][3]);
                }
        }
        const float2 w2 = *reinterpret_cast<const float2*>(&wt[now.slot][2 * t]);
        const uint32_t takes = picked.takes[now.slot] >> (2 * t);
#pragma unroll
        for (int m = 0; m < DOWN_MT; m++) {
            if (takes & 1) acc[m][0] = fmaf(w2.x, sum[m][0], acc[m][0]), acc[m][2] = fmaf(w2.x, sum[m][2], acc[m][2]);
            if (takes & 2) acc[m][1] = fmaf(w2.y, sum[m][1], acc[m][1]), acc[m][3] = fmaf(w2.y, sum[m][3], acc[m][3]);
        }
        __syncwarp();                                           // (all lanes have read the place)
        now.next(slots, nb);
        spare = at, at = at + D::SLOT == ring + DOWN_DEPTH * D::SLOT ? ring : at + D::SLOT;
    }
    __syncthreads();                                            // every ring has been copied and read: the sums lie over them
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int m = 0; m < DOWN_MT; m++) leave_sums<DOWN_MT>(red, warp, lane, m, acc[m]);
    __syncthreads();
    const int i = threadIdx.x, m = i >> 7, col = (i >> 4) & 7, f = i & 15, n = (strip0 + m) * 16 + f;
    float y = sum_of<DOWN_W, DOWN_MT>(red, m, col, f);         // (a thread an output)
    if (p.S > 1) {
        cluster_wait();
        if (rank) st_cluster_f32(mapa_cluster(smem_u32(smem) + D::BYTES + ((rank - 1) * DOWN_MT * 128 + i) * 4, 0), y);
        cluster_sync_all();
        if (rank) return;
        for (int k = 0; k < p.S - 1; k++) y += reinterpret_cast<const float*>(smem + D::BYTES)[k * DOWN_MT * 128 + i];
    }
    if (col < p.T && n < p.H) {
        if (p.out_bf16)
            ((__nv_bfloat16*)p.out)[(size_t)col * p.ldo + n] = __float2bfloat16_rn(y);
        else
            ((float*)p.out)[(size_t)col * p.ldo + n] = y;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------
Weight weight(const void* codes, const void* scales, int N, int K, int group, int pair) {
    Weight w = {};
    w.codes = (const uint4*)codes, w.scales = (const uint32_t*)scales, w.N = N, w.K = K;
    const int half = pair ? N / 2 : N;
    w.strips = (half + 15) / 16 * (pair ? 2 : 1), w.blocks = (K + 63) / 64, w.qgroups = (K + group - 1) / group;
    return w;
}

// Stages of a team beside the fragments of the rows: 0 where there is no room for two.
template <int MODE, int NT, int GROUP>
int stream_stages(int blocks) {
    const long long room = 227 * 1024 - 2048 - (MODE == GROUPED ? 8 * (GROUPS_MAX + 1) : 0) - Stream<NT, GROUP>::RED - (long long)blocks * NT * 1024;
    const long long n = room / (TEAMS * Stream<NT, GROUP>::STAGE);
    return n < 2 ? 0 : n < 5 ? (int)n : 5;
}

// max_units: the units of the launch, or more (blocks without one leave at once)
template <int MODE, int NT, int GROUP, bool PAIR>
int launch_stream(const Args& p, long long max_units, cudaStream_t stream) {
    const int stages = stream_stages<MODE, NT, GROUP>(p.w.blocks), bytes = Stream<NT, GROUP>::bytes(p.w.blocks, stages);
    auto kernel = gemm_q4_stream_kernel<MODE, NT, GROUP, PAIR>;
    static q4::SmemLimit limit;
    if (const int e = limit.lift((const void*)kernel)) return e;
    const int sms = q4::sm_count();
    return launch_pdl(kernel, dim3((unsigned)(max_units < sms ? max_units : sms)), dim3(STREAM_THREADS), (size_t)bytes, stream, p, stages);
}

// One weight, 8 NT rows (24: any number, in passes).  Streamed where a block a strip does not fit the SMs at once, three each, or, above eight rows, where there are
// 1.5 units an SM.  (us of another, a block a strip / streamed: 8 rows of 6,144 x 2,048, 384 blocks, 3.5 / 5.1, of 7,168 x 2,048, 448, 5.5 / 5.1, of 12,288 x 2,048
// 6.9 / 6.0, of 8,192 x 5,632 16.7 / 10.6, of a pair 11,264 x 2,048, 352, 4.9 / 5.9, of a pair 14,336 x 2,048, 448, 7.4 / 6.7; 16 rows of 6,144 x 2,048, 192 units, 6.3 / 7.4,
// of a pair 11,264 x 2,048, 352, 8.9 / 8.3; 24 rows of the two 8.6 / 8.8, 12.6 / 10.2.)
template <int NT, int GROUP>
int run_dense(const Args& p, bool pair, cudaStream_t stream) {
    const int half = pair ? p.w.strips / 2 : p.w.strips;
    const long long units = pair ? half : (half + 1) / 2;
    const int sms = q4::sm_count();
    if (p.M <= 8 * NT && (half > 3 * sms || (NT > 1 && 2 * units >= 3 * sms)) && stream_stages<DENSE, NT, GROUP>(p.w.blocks))
        return pair ? launch_stream<DENSE, NT, GROUP, true>(p, units, stream) : launch_stream<DENSE, NT, GROUP, false>(p, units, stream);
    return pair ? launch_pdl(gemm_q4_direct_kernel<2, NT, GROUP>, dim3(half), 256, 0, stream, p)
                : launch_pdl(gemm_q4_direct_kernel<1, NT, GROUP>, dim3(half), 256, 0, stream, p);
}

template <int GROUP>
int run_gemm(const Args& p, bool pair, cudaStream_t stream) {
    const int half = pair ? p.w.strips / 2 : p.w.strips;
    if (p.offsets) {
        const long long chunks = (long long)min(p.M, p.G) + p.M / 8;
        // Two tiles of rows at a time where groups have more than nine on average.  (us, one / two: 60 experts of a pair 2,816 x 2,048 at 8 rows an expert 61 / 63, at 10
        // 73 / 65, at 14 90 / 79; of 2,048 x 1,408 39 / 40, 45 / 42, 55 / 50.)
        if (p.M > 9 * p.G && stream_stages<GROUPED, 2, GROUP>(p.w.blocks) && chunks * half <= 0x3fffffff)
            return pair ? launch_stream<GROUPED, 2, GROUP, true>(p, chunks * half, stream)
                        : launch_stream<GROUPED, 2, GROUP, false>(p, chunks * ((half + 1) / 2), stream);
        if (!stream_stages<GROUPED, 1, GROUP>(p.w.blocks) || chunks * half > 0x3fffffff) return -1;
        if (pair) return launch_stream<GROUPED, 1, GROUP, true>(p, chunks * half, stream);
        return launch_stream<GROUPED, 1, GROUP, false>(p, chunks * ((half + 1) / 2), stream);
    }
    if (p.M <= 8) return run_dense<1, GROUP>(p, pair, stream);
    return p.M <= 16 ? run_dense<2, GROUP>(p, pair, stream) : run_dense<3, GROUP>(p, pair, stream);
}

template <int GROUP>
int run_experts(const Args& up, const DownArgs& down, cudaStream_t stream) {
    if (!stream_stages<EXPERTS, 1, GROUP>(up.w.blocks)) return -1;
    const long long pairs = (long long)up.M * up.top_k, slots = pairs < up.E ? pairs : up.E;
    const long long units = slots * (up.w.strips / 2) + (up.shared.codes ? up.shared.strips / 2 : 0);
    int e = launch_stream<EXPERTS, 1, GROUP, true>(up, units, stream);
    if (e) return e;
    static q4::SmemLimit limit;
    if ((e = limit.lift((const void*)experts_down_kernel<GROUP>))) return e;
    return launch_pdl_cluster(experts_down_kernel<GROUP>, dim3((down.down.strips + DOWN_MT - 1) / DOWN_MT, 1, down.S), dim3(DOWN_THREADS),
                              (size_t)(DownRing<GROUP>::BYTES + (down.S > 1 ? DownRing<GROUP>::PARTS : 0)), stream, down.S, down);
}

uint32_t g_wait_limit = WAIT_LIMIT_US;
int g_test_fault = 0;

}  // namespace

#define BY_GROUP(CALL)              \
    switch (group) {                \
        case 32: return CALL(32);   \
        case 64: return CALL(64);   \
        case 128: return CALL(128); \
    }                               \
    return (int)cudaErrorInvalidValue

// x: [M, K] bfloat16, row pitch ldx; codes, scales: a weight of G groups of N rows (a pair's: both halves) and K columns; out: [M, N] (a pair:
// [M, N / 2] act(gate) * up) float32 or bfloat16, row pitch ldo; offsets: null (G must be 1) or [G + 1], rows [offsets[g], offsets[g + 1]) meet group g.
// early: the weight may be read before what is in front of this launch has ended.
// Returns -1, with nothing launched, for more than 1,024 groups, or groups of rows that shared memory does not hold (K beyond 5,500 or so).
MOE_API int moe_gemm_q4(const void* x, int ldx, int M, const void* codes, const void* scales, int G, int N, int K, int group, int pair, void* out,
                        int out_bf16, int ldo, const float* bias, const int* offsets, int act, float act_param, int early, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !codes || !scales || !out || K <= 0 || G <= 0 || (G > 1 && !offsets) || (pair && N % 2)) return (int)cudaErrorInvalidValue;
    if (G > GROUPS_MAX) return -1;
    Args p = {};
    p.w = weight(codes, scales, N, K, group, pair);
    p.x = (const __nv_bfloat16*)x, p.ldx = ldx, p.M = M, p.vec = K % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & 7) == 0;
    p.out = out, p.out_bf16 = out_bf16, p.ldo = ldo, p.bias = bias, p.offsets = offsets, p.G = G, p.N = pair ? N / 2 : N;
    p.act = act, p.act_param = act_param, p.early = early, p.bits = q4::bits(), p.waits = q4::Waits{status, g_wait_limit, g_test_fault};
#define GO(GR) run_gemm<GR>(p, pair != 0, stream)
    BY_GROUP(GO);
#undef GO
}

// x: [T, H] bfloat16, row pitch ldx; idx, wk: [T, top_k]; gate: [T] or null; gu [E, 2 size, H] and sgu [2 shared, H] pairs, down [E, H, size], sdown
// [H, shared]; shared 0: no shared expert; scratch: 3 KB for each 64 features of the experts that may be picked
// (min(T top_k, E)) and of the shared one; early: as above (the second kernel reads its weights early in any case: the first has waited for what
// wrote them).  Returns -1 for what it does not take: more than 8 tokens, 1,024 experts or 128 picks, rows that shared
// memory does not hold (H beyond 6,000 or so).
MOE_API int moe_experts_q4(const void* x, int ldx, int T, int H, const int* idx, const float* wk, int top_k, int E, int size, const void* gu_codes,
                           const void* gu_scales, const void* down_codes, const void* down_scales, int shared, const void* sgu_codes,
                           const void* sgu_scales, const void* sdown_codes, const void* sdown_scales, const float* gate, int group, void* scratch,
                           long long scratch_bytes, void* out, int out_bf16, int ldo, int early, int* status, cudaStream_t stream) {
    if (T <= 0 || H <= 0) return 0;
    if (T > FEW || E > EXPERTS_MAX || (long long)T * top_k > PAIRS_MAX) return -1;
    if (!x || !idx || !wk || !scratch || !out || E <= 0 || top_k <= 0 || size <= 0 || ((uintptr_t)scratch & 15) || (shared > 0 && (!sgu_codes || !sdown_codes)))
        return (int)cudaErrorInvalidValue;
    Args up = {};
    DownArgs d = {};
    up.x = (const __nv_bfloat16*)x, up.ldx = ldx, up.vec = H % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & 7) == 0, up.M = T;
    up.idx = idx, up.top_k = top_k, up.E = E, up.early = early, up.bits = q4::bits(), up.waits = q4::Waits{status, g_wait_limit, g_test_fault};
    up.w = weight(gu_codes, gu_scales, 2 * size, H, group, 1), d.down = weight(down_codes, down_scales, H, size, group, 0);
    if (shared > 0) up.shared = weight(sgu_codes, sgu_scales, 2 * shared, H, group, 1), d.shared = weight(sdown_codes, sdown_scales, H, shared, group, 0);
    const long long slots = (long long)T * top_k < E ? (long long)T * top_k : E;
    up.frag = (uint8_t*)scratch, up.frag_blocks = d.down.blocks, up.sfrag = up.frag + slots * d.down.blocks * TERMS_BLOCK;
    if (scratch_bytes < (slots * d.down.blocks + (shared + 63) / 64) * TERMS_BLOCK) return (int)cudaErrorInvalidValue;
    d.frag = up.frag, d.sfrag = up.sfrag, d.bits = up.bits;
    d.T = T, d.H = H, d.E = E, d.top_k = top_k, d.idx = idx, d.wk = wk, d.gate = gate, d.out = out, d.out_bf16 = out_bf16, d.ldo = ldo;
    // blocks of a cluster: one block an SM, but five blocks of 64 k a warp are done sooner than two cluster barriers
    const long long most = slots * d.down.blocks + (shared > 0 ? d.shared.blocks : 0);
    d.S = most <= 5 * DOWN_W ? 1 : max(1, min(8, q4::sm_count() / ((d.down.strips + DOWN_MT - 1) / DOWN_MT)));
#define GO(GR) run_experts<GR>(up, d, stream)
    BY_GROUP(GO);
#undef GO
}

// Whether shared memory holds what groups of few rows need of rows of K elements (layer: what the first kernel of a layer of experts needs).
MOE_API int moe_q4_holds_rows(int K, int group, int layer) {
    const int blocks = (K + 63) / 64;
#define GO(GR) (layer ? stream_stages<EXPERTS, 1, GR>(blocks) : stream_stages<GROUPED, 1, GR>(blocks)) > 0
    BY_GROUP(GO);
#undef GO
}

void q4::few_rows_wait_test(int fault, uint32_t wait_limit) { g_test_fault = fault, g_wait_limit = wait_limit; }
