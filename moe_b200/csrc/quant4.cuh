// Weights held in 4 bits, as every kernel that reads them sees them.
//
// W [G, N, K]: `group` (32, 64 or 128) neighbouring k of a row share a scale s of five significant bits, and an element is q s with
// a whole number q, -7 <= q <= 7.  q has three bits, s five, so q s IS a bfloat16: every product of such a weight, whether the
// values are formed in front of the tensor core or the scale is applied behind it, is a product of the same numbers.
//
// Rows come in strips of 16, k in blocks of 64.  A block of a strip is 512 bytes of codes, 16 for each lane of a warp: lane 4 r + t
// holds rows r and r + 8 at k = 16 j + 4 t + {0, 1, 2, 3} in its 32-bit word j.  Those are the A fragment of an m16n8k16 product whose
// k are taken in the order of the fragment (the B operand's are permuted alike: a lane's four k of 16 are neighbours, one 8-byte
// load or store).  Word j, low to high: four times 4 bits of the first k of a pair (rows r, r + 8 at k 4 t; rows r, r + 8 at 4 t + 2), then the same of the second (4 t + 1, 4 t + 3), each q + 8.
//   codes   [G][strips][ceil(K / 64)][32][16 bytes]
//   scales  [G][strips][ceil(K / group)][8][2] bfloat16: rows r and r + 8 beside one another
// Rows beyond N have scale 0, k beyond K q = 0.  A pair (gate rows and up rows, N / 2 each) fills whole strips with either half.
#pragma once
#include "common.cuh"

namespace q4 {

constexpr int STRIP = 16;

struct Weight {
    const uint4* codes;            // [G][strips][blocks][32]
    const uint32_t* scales;        // [G][strips][qgroups][8], a pair of bfloat16 each
    int strips, blocks, qgroups;   // of one group
    int N, K;                      // rows (of both halves of a pair) and k
};

// The eight elements of a word as bfloat16 pairs, a[0..3] the fragment's registers: 0x4300 | n is 128 + n, less 136 is q, exactly.  The
// mask and the exponent come as kernel arguments: (w & mask) | exponent is then ONE instruction (with both as literals it is two, and
// the logic unit is what bounds these kernels).
struct Bits {
    uint32_t mask, exponent;
};
inline Bits bits() { return Bits{0x000f000fu, 0x43004300u}; }
__device__ __forceinline__ void unpack(uint32_t w, const Bits& k, uint32_t (&a)[4]) {
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t v;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w >> (4 * i)), "r"(k.mask), "r"(k.exponent));
        const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
        a[i] = *reinterpret_cast<const uint32_t*>(&q);
    }
}
__device__ __forceinline__ float scale_lo(uint32_t s) { return __uint_as_float(s << 16); }            // row r
__device__ __forceinline__ float scale_hi(uint32_t s) { return __uint_as_float(s & 0xffff0000u); }    // row r + 8

// a[i] *= the scale of its row, exactly
__device__ __forceinline__ void scale(uint32_t (&a)[4], uint32_t s) {
    const uint32_t lo = __byte_perm(s, 0, 0x1010), hi = __byte_perm(s, 0, 0x3232);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t m = (i & 1) ? hi : lo;
        const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a[i]), *reinterpret_cast<const __nv_bfloat162*>(&m));
        a[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// D = A B + C of one 16 x 16 tile of weights and eight columns of tokens
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// Scales of a block of 64 k: two where a group is 32, one otherwise (the same for two blocks where it is 128).
template <int GROUP>
struct Scales {
    static constexpr int N = GROUP == 32 ? 2 : 1;
    uint32_t s[N];
    __device__ __forceinline__ void load(const uint32_t* strip, int block, int qgroups, int r) {      // strip: scales of the strip
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int q = GROUP == 32 ? 2 * block + i : GROUP == 64 ? block : block >> 1;
            s[i] = q < qgroups ? __ldg(strip + (size_t)q * 8 + r) : 0u;
        }
    }
};

// ---- barriers and bulk copies ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false: the barrier did not complete within limit_us (the site is recorded), or another role of the block gave up
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t limit_us, int* status, int site) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = global_ns();
    for (uint32_t i = 1;; i++) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 31u) == 0) {
            if (abort_flag && *abort_flag) return false;
            if (global_ns() - t0 > (unsigned long long)limit_us * 1000ull) break;
        }
    }
    wait_ran_out(status, site);
    return false;
}
// `bytes` (a multiple of 16) from global memory, counted by a barrier of this block
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts8(uint32_t a, uint2 v) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory"); }

// Limits and faults of the waits, set for all kernels of the library by moe_q4_set_wait_test.
struct Waits {
    int* status;
    uint32_t limit_us;
    int test_fault;
};

// ---- host -------------------------------------------------------------------------------------------------------------------------------
constexpr int DEVICES = 64;
inline int device() {
    int d = 0;
    return cudaGetDevice(&d) == cudaSuccess && d >= 0 && d < DEVICES ? d : DEVICES;
}
// SMs of the current device
inline int sm_count() {
    static int known[DEVICES + 1];
    const int d = device();
    if (!known[d]) {
        int n = 0;
        known[d] = d < DEVICES && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d) == cudaSuccess ? n : 148;
    }
    return known[d];
}
// Lets a kernel have all the dynamic shared memory that a block may have, once a device (each has its own copy of the kernel; two threads that come first
// set the same).
struct SmemLimit {
    bool done[DEVICES + 1] = {};
    int lift(const void* kernel) {
        const int d = device();
        if (d < DEVICES && done[d]) return 0;
        int most = 0;
        cudaFuncAttributes a;
        cudaError_t e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, d);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, kernel);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)a.sharedSizeBytes);
        if (e == cudaSuccess) done[d] = true;
        return (int)e;
    }
};

void few_rows_wait_test(int fault, uint32_t wait_limit);      // gemm_q4.cu

}  // namespace q4
