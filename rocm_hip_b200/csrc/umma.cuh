// umma.cuh -- the fifth-generation tensor cores as the attention kernels use them: one thread issues tcgen05.mma on
// operands that the copy engine (TMA) placed in shared memory, or on an A operand in tensor memory; accumulators stay
// in tensor memory, whose lane i is row i of a 128-row tile, and come to registers by tcgen05.ld. Waits are bounded
// (mbar_wait): a role that gives up marks the CTA dead, everything after that is skipped, and the kernel ends.

#ifndef B200_UMMA_CUH
#define B200_UMMA_CUH

#include <cuda.h>

#include <type_traits>

#include "common.cuh"

namespace b200 {

constexpr int TILE_ROWS = 128;
constexpr int CHUNK = 64;                                // 16-bit values in a 128-byte swizzled row
constexpr int CHUNK_BYTES = TILE_ROWS * CHUNK * 2;       // [128 rows][64 values]

// ---- shared-memory operands, 128-byte swizzle: 8 rows of 128 bytes are an atom of 1024 bytes. A descriptor's upper half is
// the same for all of them; the lower half is the address and, for MN-major ones, the way to the next 64 values.
// K-major (rows of 64 values along the contraction): the atoms of further rows follow at 1024 bytes.
// MN-major (rows along the contraction, 64 values of the other axis each): eight more rows follow at 1024 bytes, the next
// 64 values of a row at CHUNK_BYTES.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(unsigned smem) { return ((smem & 0x3ffff) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn_major(unsigned smem) { return ((smem & 0x3ffff) >> 4) | ((uint32_t)(CHUNK_BYTES >> 4) << 16); }

// 16-bit operands (both fp16 or both bf16), fp32 accumulator, M = 128
template <typename T>
__device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
    const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// One thread of a converged warp. The instruction takes its operands from the warp's uniform registers: issued from code
// that all lanes run, they are computed there; from a branch that a single lane took, each had to be moved over first
// (100 clocks an instruction and more).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// D[128 x n] (+)= A[128 x 16] B[16 x n], A and B in shared memory (lower halves of their descriptors)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(DESC_HI)
                 : "memory");
}
// the same with A in tensor memory (16-bit pairs, one column per pair)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(DESC_HI)
                 : "memory");
}
// arrives on the barrier once everything this thread has issued to the tensor cores is done
__device__ __forceinline__ void mma_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, int cols) {   // one warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int cols) {     // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}

#define R32_(x, c) "=r"(x[c]), "=r"(x[c + 1]), "=r"(x[c + 2]), "=r"(x[c + 3]), "=r"(x[c + 4]), "=r"(x[c + 5]), "=r"(x[c + 6]), "=r"(x[c + 7])
#define P32_(x, c) "+r"(x[c]), "+r"(x[c + 1]), "+r"(x[c + 2]), "+r"(x[c + 3]), "+r"(x[c + 4]), "+r"(x[c + 5]), "+r"(x[c + 6]), "+r"(x[c + 7])
#define S32_(x, c) "r"(x[c]), "r"(x[c + 1]), "r"(x[c + 2]), "r"(x[c + 3]), "r"(x[c + 4]), "r"(x[c + 5]), "r"(x[c + 6]), "r"(x[c + 7])
#define L32_ "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"
#define L32_1_ "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32}"

// 32 columns of this warp's 32 lanes: thread i gets lane i's. The values may be used after tmem_ld_wait and tmem_pin.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " L32_ ", [%32];"
                 : R32_(x, 0), R32_(x, 8), R32_(x, 16), R32_(x, 24)
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// keeps the compiler from using the registers before this point
__device__ __forceinline__ void tmem_pin(uint32_t* x) { asm volatile("" : P32_(x, 0), P32_(x, 8), P32_(x, 16), P32_(x, 24)); }
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], " L32_1_ ";" ::"r"(addr), S32_(x, 0), S32_(x, 8), S32_(x, 16), S32_(x, 24)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- copies: a box of a tensor map to shared memory, bytes counted on the barrier
__device__ __forceinline__ void mbar_expect(unsigned long long* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// 2^x to 22 bits; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the largest of three; a NaN among numbers is passed over
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x of a pair on the FMA pipe, for x up to 127: x = n + f with n = floor(x) (adding 1.5 2^23 rounded down leaves n in the low
// mantissa bits), 2^f by the polynomial of degree DEG that has the least relative error on [0, 1] among those that are
// 1 at 0 (degree 3: 8.6e-5, degree 4: 3.0e-6; a linear programme's solution), times 2^n put together from its bits. x below -127
// (and -inf) gives exactly 0, NaN gives NaN. Eleven or twelve instructions on pipes that a softmax leaves idle, against
// two on the special-function unit, which it keeps busiest.
template <int DEG>
__device__ __forceinline__ f2 ex2_poly(f2 x) {
    float a, b;
    upk2(x, a, b);
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(a));     // -127
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(b));
    x = pk2(a, b);
    const f2 magic = pk2(12582912.0f, 12582912.0f);
    f2 r;
    asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(magic));
    const f2 f = sub2(x, sub2(r, magic));
    f2 y;
    if constexpr (DEG == 3) {
        y = fma2(pk2(0.07706713676452637f, 0.07706713676452637f), f, pk2(0.22764486074447632f, 0.22764486074447632f));
        y = fma2(y, f, pk2(0.6951168179512024f, 0.6951168179512024f));
    } else {
        y = fma2(pk2(0.013427390716969967f, 0.013427390716969967f), f, pk2(0.05224123224616051f, 0.05224123224616051f));
        y = fma2(y, f, pk2(0.24128079414367676f, 0.24128079414367676f));
        y = fma2(y, f, pk2(0.6930447816848755f, 0.6930447816848755f));
    }
    y = fma2(y, f, pk2(1.0f, 1.0f));
    const uint32_t n0 = ((uint32_t)r << 23) + 0x3f800000u, n1 = ((uint32_t)(r >> 32) << 23) + 0x3f800000u;
    return mul2(y, pk2(__uint_as_float(n0), __uint_as_float(n1)));
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack_bf16(lo, hi);
    else return pack_f16(lo, hi);
}

// v 2^e for |e| < 250, exact but where the result is subnormal (two multiplications; ldexpf is twenty instructions)
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float scale2e(float v, int e) { return v * pow2(e / 2) * pow2(e - e / 2); }
// v as fp16 hi (+ lo)
__device__ __forceinline__ void split16(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = pack_f16(a - f.x, b - f.y);
}

}  // namespace b200

#endif  // B200_UMMA_CUH
