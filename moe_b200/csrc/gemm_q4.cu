// Products of few rows over weights held in 4 bits (the format: quant4.cuh), and a layer of routed experts of few tokens.
//
//   y[m, n] = sum_k x[m, k] q[n, k] s[n, k / group] (+ b[n]), or act(gate) * up of a pair's two rows.
//
// What bounds them is the stream of codes, 0.53 bytes an element, and close behind it the issue slots: 6.5 TB/s are 46 elements a cycle and
// SM.  So an element costs about two thirds of an instruction: the weights are the A operand of m16n8k16 products straight from the registers
// that they were loaded to (two shifts, masks and subtractions a pair of elements, no shared memory), a product takes eight rows of x for the price of
// one, and the scale is applied to the sums of a group's 64 k (four products from zero, then one multiply-add an output), which also keeps
// the sums in plain 32-bit additions but for those 64.  A warp takes every W-th block of 64 k of its strip, so a block of W warps reads
// W * 512 neighbouring bytes; D blocks a warp are in flight, the first ones asked for before the wait on the predecessor.  The warps'
// sums are added up through shared memory in the order of the warps.
#include "quant4.cuh"

namespace {

using q4::Weight;

struct Rows {
    const __nv_bfloat16* x;        // [M, K], pitch ldx
    int ldx, vec;                  // vec: rows of whole 8-byte units
};

// The four B registers pairs of a block of 64 k for the lane's row (null: zeros)
__device__ __forceinline__ void load_rows(const __nv_bfloat16* row, int k0, int K, int vec, int t, uint2 (&b)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int k = k0 + 16 * j + 4 * t;
        b[j] = make_uint2(0u, 0u);
        if (!row) continue;
        if (vec) {
            if (k < K) b[j] = *reinterpret_cast<const uint2*>(row + k);
        } else {
            uint32_t e[4];
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] = k + i < K ? (uint32_t)__bfloat16_as_ushort(row[k + i]) : 0u;
            b[j] = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
        }
    }
}

// acc += one block of 64 k of MT strips against NT tiles of eight rows
template <int MT, int NT, int GROUP>
__device__ __forceinline__ void block_product(const uint4 (&code)[MT], const q4::Scales<GROUP> (&sc)[MT], const uint2 (&b)[NT][4], float (&acc)[MT][NT][4]) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < q4::Scales<GROUP>::N; h++) {
            constexpr int WORDS = 4 / q4::Scales<GROUP>::N;
            float c[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                uint32_t a[4];
                q4::unpack(q4::word(code[m], h * WORDS + i), a);
#pragma unroll
                for (int n = 0; n < NT; n++) q4::mma(c[n], a, b[n][h * WORDS + i]);
            }
            const float lo = q4::scale_lo(sc[m].s[h]), hi = q4::scale_hi(sc[m].s[h]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                acc[m][n][0] = fmaf(lo, c[n][0], acc[m][n][0]), acc[m][n][1] = fmaf(lo, c[n][1], acc[m][n][1]);
                acc[m][n][2] = fmaf(hi, c[n][2], acc[m][n][2]), acc[m][n][3] = fmaf(hi, c[n][3], acc[m][n][3]);
            }
        }
}

// The sums of W warps, added up in order: red [W][MT][8 NT][16 + 1]; thread i gets output i of MT * 8 NT * 16 (rows of the strip fastest)
template <int MT, int NT>
__device__ __forceinline__ void leave_sums(float* red, int warp, int lane, const float (&acc)[MT][NT][4]) {
    const int r = lane >> 2, t = lane & 3;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                red[((warp * MT + m) * 8 * NT + 8 * n + 2 * t + (i & 1)) * 17 + r + 8 * (i >> 1)] = acc[m][n][i];
}
template <int W, int MT, int NT>
__device__ __forceinline__ float sum_of(const float* red, int m, int col, int row) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) v += red[((w * MT + m) * 8 * NT + col) * 17 + row];
    return v;
}

struct GemmArgs {
    Weight w;
    Rows rows;
    void* out;
    int out_bf16, ldo;
    const float* bias;
    const int* offsets;            // null: one group of M rows
    int M, N;                      // N: output features (of a pair: of one half)
    int act;
    float act_param;
};

constexpr int DEPTH = 4;           // blocks of a warp in flight

// Grid: (strips of the output, groups, 1).  MT 2: a pair's gate and up strip.
template <int W, int MT, int NT, int GROUP>
__global__ void __launch_bounds__(W * 32)
gemm_q4_kernel(const __grid_constant__ GemmArgs p) {
    __shared__ float red[W * MT * 8 * NT * 17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int strip = blockIdx.x, g = blockIdx.y, blocks = p.w.blocks;
    const uint4* codes[MT];
    const uint32_t* scales[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const size_t s = (size_t)g * p.w.strips + strip + m * (p.w.strips / 2);
        codes[m] = p.w.codes + s * blocks * 32 + lane;
        scales[m] = p.w.scales + s * p.w.qgroups * 8;
    }
    int row0 = 0, row_end = p.M;
    bool waited = false;
    if (p.offsets) {                                     // (written by an earlier kernel, maybe the predecessor)
        pdl_sync();
        waited = true;
        row0 = max(0, p.offsets[g]), row_end = min(p.M, p.offsets[g + 1]);
        if (row0 >= row_end) return;
    }
    for (; row0 < row_end; row0 += 8 * NT) {
        uint4 code[DEPTH][MT];
        q4::Scales<GROUP> sc[DEPTH][MT];
        float acc[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
        auto load = [&](int d, int b) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
                code[d][m] = q4::ld_codes(codes[m] + (size_t)b * 32);
                sc[d][m].load(scales[m], b, p.w.qgroups, r);
            }
        };
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (warp + d * W < blocks) load(d, warp + d * W);
        if (!waited) pdl_sync();
        waited = true;
        const __nv_bfloat16* xr[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) xr[n] = row0 + 8 * n + r < row_end ? p.rows.x + (size_t)(row0 + 8 * n + r) * p.rows.ldx : nullptr;
        for (int b0 = warp; b0 < blocks; b0 += DEPTH * W) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                const int b = b0 + d * W;
                if (b >= blocks) break;
                uint2 x[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++) load_rows(xr[n], b * 64, p.w.K, p.rows.vec, t, x[n]);
                block_product<MT, NT, GROUP>(code[d], sc[d], x, acc);
                if (b + DEPTH * W < blocks) load(d, b + DEPTH * W);
            }
        }
        leave_sums<MT, NT>(red, warp, lane, acc);
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * NT * 16; i += W * 32) {
            const int col = i >> 4, f = i & 15, n = strip * 16 + f, row = row0 + col;
            if (n >= p.N || row >= row_end) continue;
            float v = sum_of<W, MT, NT>(red, 0, col, f);
            if (MT == 2)
                v = glu_mul(p.act, p.act_param, v, sum_of<W, MT, NT>(red, MT - 1, col, f));
            else
                v = plain_act(p.act, p.bias ? v + p.bias[n] : v);
            if (p.out_bf16)
                ((__nv_bfloat16*)p.out)[(size_t)row * p.ldo + n] = __float2bfloat16_rn(v);
            else
                ((float*)p.out)[(size_t)row * p.ldo + n] = v;
        }
        __syncthreads();
    }
}

// ---- a layer of routed experts of few tokens -----------------------------------------------------------------------------------------
//   out_t = sum_e w_te Wd_e a_te + gate_t Wd_s a_t,  a = silu(Wg h_t) * (Wu h_t),  w_te the sum of t's weights for expert e
// in two launches.  The eight columns of a product are the step's tokens whatever the expert, so that nothing is gathered: an expert's
// block forms all tokens' rows and keeps those of the tokens that picked it, and the second product takes zeros for the others.  Both
// kernels find the list of picked experts (in order of their numbers) from the picks themselves.  The second takes one strip of the output through
// ALL picked experts and the shared one, w_te on the sums of each block: nothing is left to combine.
constexpr int EXPERTS_MAX = 1024, FEW = 8, PAIRS_MAX = 512;

struct LayerArgs {
    const __nv_bfloat16* x;        // [T, H], pitch ldx
    int ldx, vec, T, H, E, top_k;
    const int* idx;                // [T, top_k]; -1: none
    const float* wk;               // [T, top_k]
    const float* gate;             // [T] or null (1)
    Weight gu, down, sgu, sdown;   // sgu.codes null: no shared expert
    __nv_bfloat16* act;            // [slots][8][pitch]
    __nv_bfloat16* sact;           // [8][spitch]
    int pitch, spitch;             // whole strips
    void* out;
    int out_bf16, ldo;
    int* status;
};

// The picked experts' bits, and the number of those below each word.  By all threads; ends with a barrier.
struct Picked {
    uint32_t bits[EXPERTS_MAX / 32];
    int before[EXPERTS_MAX / 32 + 1];
    int idx[PAIRS_MAX];
};
__device__ __forceinline__ void find_picked(const LayerArgs& p, Picked& s, bool tell) {
    const int pairs = p.T * p.top_k;
    for (int i = threadIdx.x; i < EXPERTS_MAX / 32; i += blockDim.x) s.bits[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        int e = p.idx[i];
        if (e < 0 || e >= p.E) {
            if (e != -1 && tell && p.status) atomicOr(p.status, ST_BAD_EXPERT);
            e = -1;
        } else
            atomicOr(&s.bits[e >> 5], 1u << (e & 31));
        s.idx[i] = e;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int n = __popc(s.bits[threadIdx.x]);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int)threadIdx.x >= o) upto += v;
        }
        s.before[threadIdx.x] = upto - n;
        if (threadIdx.x == 31) s.before[32] = upto;
    }
    __syncthreads();
}
// the slot-th picked expert
__device__ __forceinline__ int expert_of(const Picked& s, int slot) {
    int w = 0;
    while (s.before[w + 1] <= slot) w++;
    return w * 32 + (int)__fns(s.bits[w], 0, slot - s.before[w] + 1);
}

template <int W, int GROUP>
__global__ void __launch_bounds__(W * 32)
experts_up_kernel(const __grid_constant__ LayerArgs p) {
    __shared__ float red[W * 2 * 8 * 17];
    __shared__ Picked picked;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int shared_strips = p.sgu.codes ? p.sgu.strips / 2 : 0;
    const bool shared = (int)blockIdx.x < shared_strips;
    Weight w;
    int strip, slot = 0;
    size_t first = 0;
    if (shared) {
        w = p.sgu, strip = blockIdx.x;
    } else {
        pdl_sync();
        find_picked(p, picked, (int)blockIdx.x == shared_strips);
        const int u = blockIdx.x - shared_strips;
        w = p.gu, slot = u / (w.strips / 2), strip = u - slot * (w.strips / 2);
        if (slot >= picked.before[32]) return;
        first = (size_t)expert_of(picked, slot) * w.strips;
    }
    const int blocks = w.blocks;
    const uint4* codes[2];
    const uint32_t* scales[2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const size_t s = first + strip + m * (w.strips / 2);
        codes[m] = w.codes + s * blocks * 32 + lane;
        scales[m] = w.scales + s * w.qgroups * 8;
    }
    uint4 code[DEPTH][2];
    q4::Scales<GROUP> sc[DEPTH][2];
    float acc[2][1][4] = {};
    auto load = [&](int d, int b) {
#pragma unroll
        for (int m = 0; m < 2; m++) {
            code[d][m] = q4::ld_codes(codes[m] + (size_t)b * 32);
            sc[d][m].load(scales[m], b, w.qgroups, r);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (warp + d * W < blocks) load(d, warp + d * W);
    if (shared) pdl_sync();
    const __nv_bfloat16* xr = r < p.T ? p.x + (size_t)r * p.ldx : nullptr;
    for (int b0 = warp; b0 < blocks; b0 += DEPTH * W) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int b = b0 + d * W;
            if (b >= blocks) break;
            uint2 x[1][4];
            load_rows(xr, b * 64, w.K, p.vec, t, x[0]);
            block_product<2, 1, GROUP>(code[d], sc[d], x, acc);
            if (b + DEPTH * W < blocks) load(d, b + DEPTH * W);
        }
    }
    leave_sums<2, 1>(red, warp, lane, acc);
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * 16; i += W * 32) {
        const int col = i >> 4, f = i & 15;
        if (col >= p.T) continue;
        const float v = glu_mul(ACT_SILU, 0.f, sum_of<W, 2, 1>(red, 0, col, f), sum_of<W, 2, 1>(red, 1, col, f));
        // (rounded once, as what every product over weights of these reads)
        __nv_bfloat16* a = shared ? p.sact + (size_t)col * p.spitch : p.act + ((size_t)slot * FEW + col) * p.pitch;
        a[strip * 16 + f] = __float2bfloat16_rn(v);
    }
}

template <int W, int GROUP>
__global__ void __launch_bounds__(W * 32)
experts_down_kernel(const __grid_constant__ LayerArgs p) {
    __shared__ float red[W * 8 * 17];
    __shared__ Picked picked;
    __shared__ __align__(16) float wt[PAIRS_MAX + 1][FEW];   // a slot's weight of each token; the last one's: the shared expert's gate
    __shared__ uint32_t takes[PAIRS_MAX + 1];         // the tokens that picked it
    __shared__ short expert[PAIRS_MAX];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, strip = blockIdx.x;
    // The picks were written at least two kernels ago (this one's predecessor let it in behind its own wait): they, and the weights, are
    // read before the wait.
    find_picked(p, picked, false);
    const int slots = picked.before[32];
    for (int i = threadIdx.x; i < slots; i += W * 32) {
        const int e = expert_of(picked, i);
        expert[i] = (short)e;
        uint32_t m = 0;
        for (int c = 0; c < p.T; c++) {
            float v = 0.f;
            for (int j = 0; j < p.top_k; j++)
                if (picked.idx[c * p.top_k + j] == e) v += p.wk[c * p.top_k + j], m |= 1u << c;
            wt[i][c] = v;
        }
        for (int c = p.T; c < FEW; c++) wt[i][c] = 0.f;
        takes[i] = m;
    }
    if (threadIdx.x < FEW) wt[slots][threadIdx.x] = (int)threadIdx.x < p.T && p.sdown.codes ? (p.gate ? p.gate[threadIdx.x] : 1.f) : 0.f;
    if (threadIdx.x == FEW) takes[slots] = (1u << p.T) - 1;
    __syncthreads();
    const int nb = p.down.blocks, total = slots * nb + (p.sdown.codes ? p.sdown.blocks : 0);
    auto where = [&](int i, int* slot, int* b) {
        *slot = min(i / nb, slots), *b = i - *slot * nb;
    };
    uint4 code[DEPTH][1];
    q4::Scales<GROUP> sc[DEPTH][1];
    auto load = [&](int d, int i) {
        int slot, b;
        where(i, &slot, &b);
        const Weight& w = slot < slots ? p.down : p.sdown;
        const size_t s = (size_t)(slot < slots ? expert[slot] : 0) * w.strips + strip;
        code[d][0] = q4::ld_codes(w.codes + (s * w.blocks + b) * 32 + lane);
        sc[d][0].load(w.scales + s * w.qgroups * 8, b, w.qgroups, r);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (warp + d * W < total) load(d, warp + d * W);
    pdl_sync();
    float acc[1][1][4] = {};
    for (int i0 = warp; i0 < total; i0 += DEPTH * W) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int i = i0 + d * W;
            if (i >= total) break;
            int slot, b;
            where(i, &slot, &b);
            uint2 x[1][4];
            const bool mine = (takes[slot] >> r) & 1;
            const __nv_bfloat16* row = slot < slots ? p.act + ((size_t)slot * FEW + r) * p.pitch : p.sact + (size_t)r * p.spitch;
            load_rows(mine ? row : nullptr, b * 64, slot < slots ? p.pitch : p.spitch, 1, t, x[0]);
            float part[1][1][4] = {};
            block_product<1, 1, GROUP>(code[d], sc[d], x, part);
            const float2 w2 = *reinterpret_cast<const float2*>(&wt[slot][2 * t]);
            acc[0][0][0] = fmaf(w2.x, part[0][0][0], acc[0][0][0]), acc[0][0][1] = fmaf(w2.y, part[0][0][1], acc[0][0][1]);
            acc[0][0][2] = fmaf(w2.x, part[0][0][2], acc[0][0][2]), acc[0][0][3] = fmaf(w2.y, part[0][0][3], acc[0][0][3]);
            if (i + DEPTH * W < total) load(d, i + DEPTH * W);
        }
    }
    leave_sums<1, 1>(red, warp, lane, acc);
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * 16; i += W * 32) {
        const int col = i >> 4, f = i & 15, n = strip * 16 + f;
        if (col >= p.T || n >= p.H) continue;
        const float v = sum_of<W, 1, 1>(red, 0, col, f);
        if (p.out_bf16)
            ((__nv_bfloat16*)p.out)[(size_t)col * p.ldo + n] = __float2bfloat16_rn(v);
        else
            ((float*)p.out)[(size_t)col * p.ldo + n] = v;
    }
}

Weight weight(const void* codes, const void* scales, int N, int K, int group, int pair) {
    Weight w = {};
    w.codes = (const uint4*)codes, w.scales = (const uint32_t*)scales, w.N = N, w.K = K;
    const int half = pair ? N / 2 : N;
    w.strips = (half + 15) / 16 * (pair ? 2 : 1), w.blocks = (K + 63) / 64, w.qgroups = (K + group - 1) / group;
    return w;
}

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
MOE_API int moe_gemm_q4(const void* x, int ldx, int M, const void* codes, const void* scales, int G, int N, int K, int group, int pair, void* out,
                        int out_bf16, int ldo, const float* bias, const int* offsets, int act, float act_param, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !codes || !scales || !out || K <= 0 || G <= 0 || (G > 1 && !offsets) || (pair && N % 2) || G > 65535) return (int)cudaErrorInvalidValue;
    GemmArgs p = {};
    p.w = weight(codes, scales, N, K, group, pair);
    p.rows.x = (const __nv_bfloat16*)x, p.rows.ldx = ldx, p.rows.vec = K % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & 7) == 0;
    p.out = out, p.out_bf16 = out_bf16, p.ldo = ldo, p.bias = bias, p.offsets = offsets, p.M = M, p.N = pair ? N / 2 : N;
    p.act = act, p.act_param = act_param;
    const dim3 grid(pair ? p.w.strips / 2 : p.w.strips, G);
    constexpr int W = 8;
    const bool two = offsets ? true : M > 8;
#define GO(GR)                                                                                            \
    (pair ? (two ? launch_pdl(gemm_q4_kernel<W, 2, 2, GR>, grid, W * 32, 0, stream, p)                    \
                 : launch_pdl(gemm_q4_kernel<W, 2, 1, GR>, grid, W * 32, 0, stream, p))                   \
          : (two ? launch_pdl(gemm_q4_kernel<W, 1, 2, GR>, grid, W * 32, 0, stream, p)                    \
                 : launch_pdl(gemm_q4_kernel<W, 1, 1, GR>, grid, W * 32, 0, stream, p)))
    BY_GROUP(GO);
#undef GO
}

// bfloat16 elements of scratch that moe_experts_q4 wants
MOE_API long long moe_experts_q4_scratch(int T, int top_k, int E, int size, int shared) {
    const long long slots = (long long)T * top_k < E ? (long long)T * top_k : E;
    return slots * FEW * ((size + 15) / 16 * 16) + (long long)FEW * ((shared + 15) / 16 * 16);
}

// x: [T, H] bfloat16, row pitch ldx; idx, wk: [T, top_k]; gate: [T] or null; gu [E, 2 size, H] and sgu [2 shared, H] pairs, down [E, H, size], sdown
// [H, shared]; shared 0: no shared expert.  Returns -1 for what it does not take: more than 8 tokens, 1,024 experts or 512 picks.
MOE_API int moe_experts_q4(const void* x, int ldx, int T, int H, const int* idx, const float* wk, int top_k, int E, int size, const void* gu_codes,
                           const void* gu_scales, const void* down_codes, const void* down_scales, int shared, const void* sgu_codes,
                           const void* sgu_scales, const void* sdown_codes, const void* sdown_scales, const float* gate, int group, void* scratch,
                           void* out, int out_bf16, int ldo, int* status, cudaStream_t stream) {
    if (T <= 0 || H <= 0) return 0;
    if (T > FEW || E > EXPERTS_MAX || (long long)T * top_k > PAIRS_MAX) return -1;
    if (!x || !idx || !wk || !scratch || !out || E <= 0 || top_k <= 0 || size <= 0 || ((uintptr_t)scratch & 15) || (shared > 0 && (!sgu_codes || !sdown_codes)))
        return (int)cudaErrorInvalidValue;
    LayerArgs p = {};
    p.x = (const __nv_bfloat16*)x, p.ldx = ldx, p.vec = H % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & 7) == 0;
    p.T = T, p.H = H, p.E = E, p.top_k = top_k, p.idx = idx, p.wk = wk, p.gate = gate;
    p.gu = weight(gu_codes, gu_scales, 2 * size, H, group, 1), p.down = weight(down_codes, down_scales, H, size, group, 0);
    if (shared > 0) p.sgu = weight(sgu_codes, sgu_scales, 2 * shared, H, group, 1), p.sdown = weight(sdown_codes, sdown_scales, H, shared, group, 0);
    p.pitch = (size + 15) / 16 * 16, p.spitch = (shared + 15) / 16 * 16;
    const long long slots = (long long)T * top_k < E ? (long long)T * top_k : E;
    p.act = (__nv_bfloat16*)scratch, p.sact = p.act + slots * FEW * p.pitch;
    p.out = out, p.out_bf16 = out_bf16, p.ldo = ldo, p.status = status;
    const long long up = p.spitch / 16 + slots * (p.pitch / 16);
    if (up > 0x7fffffffll) return -1;
    auto run = [&](auto up_kernel, auto down_kernel) {
        const int e = launch_pdl(up_kernel, dim3((unsigned)up), 256, 0, stream, p);
        return e ? e : launch_pdl(down_kernel, dim3(p.down.strips), 512, 0, stream, p);
    };
#define GO(GR) run(experts_up_kernel<8, GR>, experts_down_kernel<16, GR>)
    BY_GROUP(GO);
#undef GO
}
