// Weights to 4 bits and back (the format: quant4.cuh).
//
//   s = max |w| over the group / 7, rounded to five significant bits (nearest, ties to even); q = w / s rounded (ties to even).
// s may be rounded down by 1 / 33 of itself at most, so |w| / s <= 7 (1 + 1 / 32) < 7.5 and q needs no clamp.  Decisions at a border are exact.  For
// bfloat16: max / 7 and w / s as correctly rounded 32-bit quotients, which are a border (five bits; half a step) only where the exact quotient
// is, its operands having eight and five bits.  For float32: max / 7 in 64 bits (of a 24-bit number: never nearer to a border of five bits than 2^-27 of itself
// unless on it), and w - q s, which 32 bits hold exactly, says which side of half a step w lies on.  A group whose maximum is below 7 * 2^-126 is
// held as zeros; one that holds an infinity or a NaN gets the scale NaN, so that products of it are NaN, and sets ST_NOT_FINITE.
//
// A warp takes one strip (16 rows) x 64 k (128 where a group is 128), 8 bytes a load of bfloat16, four
// lanes a 32-byte sector.  DRAM should bound both directions.  23 M weights (a pair 11,264 x 2,048, bfloat16) there and back take 25.6 us, 4.6 TB/s, with sixteen instructions an
// element there and ten back in 58 and 70 % of the issue slots: no unit is full.
#include "quant4.cuh"

namespace {

template <typename T, bool FULL>
__device__ __forceinline__ void load4(const T* row, int k, int K, bool vec, float (&v)[4]) {
    if (FULL || (vec && k + 4 <= K)) {
        if constexpr (sizeof(T) == 2) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + k));
            v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
            v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
            const float4 f = __ldg(reinterpret_cast<const float4*>(row + k));
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        }
        return;
    }
    if constexpr (!FULL)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = k + i < K ? ld_f(row + k + i) : 0.f;
}

// max / 7 to five significant bits; 0 for what is held as zeros, NaN for what is no number
template <typename T>
__device__ __forceinline__ float scale_of(float amax) {
    if (!(amax <= 3.402823466e38f)) return __uint_as_float(0x7fc00000u);
    if (amax < 0x1.cp-124f) return 0.f;                                   // 7 * 2^-126
    if constexpr (sizeof(T) == 2) {
        uint32_t u = __float_as_uint(__fdiv_rn(amax, 7.f));
        u += (1u << 18) - 1 + ((u >> 19) & 1);                            // 23 - 4 bits go
        return __uint_as_float(u & ~((1u << 19) - 1));
    }
    const double d = (double)amax / 7.0;
    unsigned long long u = (unsigned long long)__double_as_longlong(d);
    u += (1ull << 47) - 1 + ((u >> 48) & 1);                              // 52 - 4 bits go
    u &= ~((1ull << 48) - 1);
    return (float)__longlong_as_double((long long)u);
}

// w / s to the nearest whole number, ties to even, plus 8, in the low four bits
template <typename T>
__device__ __forceinline__ uint32_t code_of(float w, float s, float rs) {
    if constexpr (sizeof(T) == 2) {
        const float v = w * rs;
        return __float_as_uint(fmaf(fmaf(-v, s, w), rs, v) + 12582920.f);      // the correctly rounded quotient; 1.5 * 2^23 + 8
    }
    float q = rintf(w * rs);
    const float r = fmaf(-q, s, w), h = 0.5f * s, a = fabsf(r);           // exact: q s has eight bits and lies within a step of w
    if (a > h || (a == h && ((int)q & 1))) q += r > 0.f ? 1.f : -1.f;
    return (uint32_t)((int)q + 8);
}

// One weight's sizes, and how a block's eight warps lie: 1 << kw of them beside one another in k (units of one strip), the others in further strips.
// Grid: (units in k, strips, groups); the latter two in rounds where there are more than a grid has.
struct Shape {
    int G, N, K, pair, strips, blocks, qgroups, units, kw;
};
__device__ __forceinline__ bool row_of(const Shape& p, int strip, int r, int* row) {
    const int half = p.pair ? p.N / 2 : p.N, per = p.pair ? p.strips / 2 : p.strips;
    const int h = strip >= per ? 1 : 0, in = (strip - h * per) * q4::STRIP + r;
    *row = h * half + in;
    return in < half;
}
Shape shape_of(int G, int N, int K, int group, int pair, int span) {
    Shape s = {G, N, K, pair};
    s.strips = ((pair ? N / 2 : N) + 15) / 16 * (pair ? 2 : 1), s.blocks = (K + 63) / 64, s.qgroups = (K + group - 1) / group;
    s.units = (s.blocks + span - 1) / span;
    while (s.kw < 3 && (1 << s.kw) < s.units) s.kw++;
    return s;
}
dim3 grid_of(const Shape& s) {
    const int across = 8 >> s.kw, y = (s.strips + across - 1) / across;
    return dim3((unsigned)((s.units + (1 << s.kw) - 1) >> s.kw), (unsigned)(y < 65535 ? y : 65535), (unsigned)(s.G < 65535 ? s.G : 65535));
}

// FULL: whole strips and units, rows of whole 16-byte units: no check at a load
template <typename T, int GROUP, bool FULL>
__device__ __forceinline__ void quantize_unit(const T* __restrict__ w, const Shape& p, int g0, int strip, int u, int vec, uint4* __restrict__ codes,
                                              uint32_t* __restrict__ scales, int* status) {
    constexpr int SPAN = GROUP == 128 ? 2 : 1;                            // blocks of a unit
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, K = p.K, blocks = p.blocks, qgroups = p.qgroups;
    const size_t gs = (size_t)g0 * p.strips + strip;
    const T* wg = w + (size_t)g0 * p.N * K;
    float v[2][SPAN][16];
#pragma unroll
    for (int half = 0; half < 2; half++) {
        int row;
        const bool live = row_of(p, strip, r + 8 * half, &row) || FULL;
        const T* p_row = wg + (size_t)(live ? row : 0) * K;
#pragma unroll
        for (int b = 0; b < SPAN; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x[4];
                load4<T, FULL>(p_row, live ? (u * SPAN + b) * 64 + 16 * j + 4 * t : K, K, vec, x);
#pragma unroll
                for (int i = 0; i < 4; i++) v[half][b][4 * j + i] = x[i];
            }
    }
    constexpr int SETS = GROUP == 32 ? 2 : 1, PER = 16 * SPAN / SETS;     // scales of a unit and row, elements of this lane under one
    float s[2][SETS], rs[2][SETS], sq[2][SETS];
    bool bad = false;
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
        for (int g = 0; g < SETS; g++) {
            uint32_t m = 0;                                               // (magnitudes are ordered as their bits, infinity and NaN above all)
#pragma unroll
            for (int i = 0; i < PER; i++) m = max(m, __float_as_uint(v[half][(g * PER + i) / 16][(g * PER + i) % 16]) & 0x7fffffffu);
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            s[half][g] = scale_of<T>(__uint_as_float(m));
            bad = bad || s[half][g] != s[half][g];
            // (a group of zeros, or of no numbers: w * 0 for q, and no step)
            rs[half][g] = s[half][g] > 0.f ? 1.f / s[half][g] : 0.f, sq[half][g] = s[half][g] > 0.f ? s[half][g] : 0.f;
        }
    if (bad && status) atomicOr(status, ST_NOT_FINITE);
    if (t == 0) {
#pragma unroll
        for (int g = 0; g < SETS; g++) {
            const int q = GROUP == 32 ? 2 * u + g : u;
            if (q < qgroups)
                scales[(gs * qgroups + q) * 8 + r] = (__float_as_uint(s[0][g]) >> 16) | (__float_as_uint(s[1][g]) & 0xffff0000u);
        }
    }
#pragma unroll
    for (int b = 0; b < SPAN; b++) {
        if (u * SPAN + b >= blocks) break;
        uint32_t out[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int g = GROUP == 32 ? j / 2 : 0;
            uint32_t o = 0;
#pragma unroll
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {                             // k 4 t + i: pair i / 2, place i % 2
                    const int at = 16 * (i & 1) + 8 * (i >> 1) + 4 * half;
                    o |= (code_of<T>(v[half][b][4 * j + i], sq[half][g], rs[half][g]) << at) & (15u << at);
                }
            }
            out[j] = o;
        }
        codes[(gs * blocks + u * SPAN + b) * 32 + lane] = make_uint4(out[0], out[1], out[2], out[3]);
    }
}

// Blocks an SM: as many as the registers of a unit's elements allow with few spills (bfloat16, whole units: six, 2 us of the 26 of both directions less than
// what the compiler takes by itself).
template <typename T, int GROUP, bool FULL>
constexpr int quantize_blocks = GROUP == 128 ? 3 : FULL && sizeof(T) == 2 ? 6 : 4;
template <typename T, int GROUP, bool FULL>
__global__ void __launch_bounds__(256, (quantize_blocks<T, GROUP, FULL>))
quantize_kernel(const T* __restrict__ w, const Shape p, int vec, uint4* __restrict__ codes, uint32_t* __restrict__ scales, int* status) {
    pdl_wait();
    const int warp = threadIdx.x >> 5, u = ((int)blockIdx.x << p.kw) + (warp & ((1 << p.kw) - 1));
    if (u >= p.units) return;
    for (int g = blockIdx.z; g < p.G; g += gridDim.z)
        for (int strip = blockIdx.y * (8 >> p.kw) + (warp >> p.kw); strip < p.strips; strip += gridDim.y * (8 >> p.kw))
            quantize_unit<T, GROUP, FULL>(w, p, g, strip, u, vec, codes, scales, status);
}

template <int GROUP>
__device__ __forceinline__ void dequantize_unit(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, const Shape& p, int g0, int strip, int b,
                                                int vec, const q4::Bits& bits, __nv_bfloat16* __restrict__ out) {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, K = p.K;
    const size_t gs = (size_t)g0 * p.strips + strip;
    const uint4 c = __ldg(codes + (gs * p.blocks + b) * 32 + lane);
    q4::Scales<GROUP> sc;
    sc.load(scales + gs * p.qgroups * 8, b, p.qgroups, r);
    __nv_bfloat16* og = out + (size_t)g0 * p.N * K;
    int row[2];
    const bool live[2] = {row_of(p, strip, r, &row[0]), row_of(p, strip, r + 8, &row[1])};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t a[4];
        q4::unpack(q4::word(c, j), bits, a);
        const int k = b * 64 + 16 * j + 4 * t;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t s2 = sc.s[GROUP == 32 ? j / 2 : 0];
            const __nv_bfloat16 s = __ushort_as_bfloat16((unsigned short)(half ? s2 >> 16 : s2 & 0xffffu));
            const __nv_bfloat162 ss = __halves2bfloat162(s, s);
            __nv_bfloat162 v[2];
#pragma unroll
            for (int p = 0; p < 2; p++) v[p] = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a[half + 2 * p]), ss);      // exact
            if (!live[half]) continue;
            __nv_bfloat16* o = og + (size_t)row[half] * K + k;
            if (vec && k + 4 <= K)
                *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(v);
            else
                for (int i = 0; i < 4 && k + i < K; i++) o[i] = reinterpret_cast<const __nv_bfloat16*>(v)[i];
        }
    }
}

template <int GROUP>
__global__ void __launch_bounds__(256, 6)
dequantize_kernel(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, const Shape p, int vec, const q4::Bits bits, __nv_bfloat16* __restrict__ out) {
    pdl_wait();
    const int warp = threadIdx.x >> 5, u = ((int)blockIdx.x << p.kw) + (warp & ((1 << p.kw) - 1));
    if (u >= p.units) return;
    for (int g = blockIdx.z; g < p.G; g += gridDim.z)
        for (int strip = blockIdx.y * (8 >> p.kw) + (warp >> p.kw); strip < p.strips; strip += gridDim.y * (8 >> p.kw))
            dequantize_unit<GROUP>(codes, scales, p, g, strip, u, vec, bits, out);
}

}  // namespace

#define BY_GROUP(CALL)            \
    switch (group) {              \
        case 32: return CALL(32);   \
        case 64: return CALL(64);   \
        case 128: return CALL(128); \
    }                             \
    return (int)cudaErrorInvalidValue

// w: [G, N, K] float32 (w_dt DT_F32) or bfloat16, contiguous; codes, scales: see quant4.cuh (strips of one G: ceil(N / 16), of a pair
// 2 ceil(N / 2 / 16)).
MOE_API int moe_q4_quantize(const void* w, int w_dt, int G, int N, int K, int group, int pair, void* codes, void* scales, int* status, cudaStream_t stream) {
    if (G <= 0 || N <= 0 || K <= 0) return 0;
    if (!w || !codes || !scales || (pair && N % 2)) return (int)cudaErrorInvalidValue;
    const Shape s = shape_of(G, N, K, group > 0 ? group : 1, pair, group == 128 ? 2 : 1);
    const int vec = K % 4 == 0 && ((uintptr_t)w & 15) == 0;
    const bool full = vec && K % 128 == 0 && (pair ? N / 2 : N) % 16 == 0;
    auto go = [&](auto kernel, auto* from) { return launch_pdl(kernel, grid_of(s), 256, 0, stream, from, s, vec, (uint4*)codes, (uint32_t*)scales, status); };
#define GO(GR)                                                                                                                              \
    (w_dt == DT_BF16 ? go(full ? quantize_kernel<__nv_bfloat16, GR, true> : quantize_kernel<__nv_bfloat16, GR, false>, (const __nv_bfloat16*)w) \
                     : go(full ? quantize_kernel<float, GR, true> : quantize_kernel<float, GR, false>, (const float*)w))
    BY_GROUP(GO);
#undef GO
}

// out: [G, N, K] bfloat16, the values that the codes stand for
MOE_API int moe_q4_dequantize(const void* codes, const void* scales, int G, int N, int K, int group, int pair, void* out, cudaStream_t stream) {
    if (G <= 0 || N <= 0 || K <= 0) return 0;
    if (!out || !codes || !scales || (pair && N % 2)) return (int)cudaErrorInvalidValue;
    const Shape s = shape_of(G, N, K, group > 0 ? group : 1, pair, 1);
    const int vec = K % 4 == 0 && ((uintptr_t)out & 7) == 0;
#define GO(GR) launch_pdl(dequantize_kernel<GR>, grid_of(s), 256, 0, stream, (const uint4*)codes, (const uint32_t*)scales, s, vec, q4::bits(), (__nv_bfloat16*)out)
    BY_GROUP(GO);
#undef GO
}

// Programmatic dependent launch on or off for the kernels of this library (on by default).
MOE_API void moe_q4_set_pdl(int enabled) { g_pdl_enabled = enabled ? 1 : 0; }
