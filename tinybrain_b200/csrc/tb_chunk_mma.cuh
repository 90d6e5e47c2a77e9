// tb_chunk_mma.cuh -- fp32-accurate fp16 operands for the tensor cores, as the
// chunk attention (tb_chunk.cu) uses them.
//
// An fp32 value x with |x| < 2^15 is carried as hi + lo, hi = fp16(x) and lo =
// fp16(x - hi): |x - hi - lo| <= 2^-22 |x|, or 2^-25 where that is larger (the
// step of fp16's subnormals).  A product is then
//     x y = hi hi' + hi lo' + lo hi'   (lo lo' <= 2^-22 |x y| is left out)
// in fp32 accumulators: three kind::f16 products, twice as fast as the three
// kind::tf32 ones that would carry as much.  Operands are scaled by powers of
// two to a largest magnitude in [2^14, 2^15), so that the absolute term is at
// most 2^-39 of the largest value of its block.
//
// Operand layouts: A in tensor memory (lane = row, 32-bit column = two
// consecutive k); B in shared memory, K-major without swizzle, 8 x 16-byte core
// matrices: [rows / 8][k / 8][8 rows][8 k], LBO 128 bytes, SBO 16 k bytes.
#pragma once

#include <cuda_fp16.h>

#include "tb_tc.cuh"

namespace tb {

// kind::f16, D fp32, A and B fp16, both K-major, M = 128.
__host__ __device__ constexpr uint32_t tc_idesc_f16(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B^T for one K = 16 step; issued by a single thread.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t dtmem, uint32_t atmem, uint64_t bdesc, uint32_t idesc,
                                              bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(dtmem),
        "r"(atmem), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// D = (A_hi + A_lo) (B_hi + B_lo)^T without lo lo, N columns, K deep.  A in
// tensor memory: k step s (16 k, 8 columns) of the high half at a + step(s), of
// the low half lo_at columns further.  B: N x K halves of 2 N K bytes each.
// The accumulator is fp32 with truncated sums (measured: each step loses 2^-25
// of it on average), so the two small products come first, while it is small,
// and nothing is carried from one call to the next: that sum is made outside,
// rounded to nearest.
template <int N, int K, class Step>
__device__ __forceinline__ void tc_mma_split(uint32_t d, uint32_t a, Step step, uint32_t lo_at, uint32_t b_hi,
                                             uint32_t b_lo) {
    constexpr uint32_t idesc = tc_idesc_f16(N);
#pragma unroll 1
    for (int product = 0; product < 3; ++product) {
        const uint32_t half = product == 0 ? lo_at : 0, b = product == 1 ? b_lo : b_hi;
#pragma unroll
        for (int s = 0; s < K / 16; ++s)
            tc_mma_f16_ts(d, a + half + step(s), tc_sdesc(b + 256 * s, 128, 16 * K), idesc, product + s > 0);
    }
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// 16 lanes x 8 N columns: a thread holds, of every 8 columns, two neighbouring ones
// (2 (lane % 4) and the next) of TMEM lane `lane / 4` and the same of lane / 4 + 8.
template <int N>
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&v)[4 * N]) {
    if constexpr (N == 4) {
        asm volatile(
            "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
            "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
            "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
            "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
            : "memory");
    } else if constexpr (N == 2) {
        asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                     "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    } else {
        static_assert(N == 1, "columns");
        asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                     "r"(v[2]), "r"(v[3])
                     : "memory");
    }
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}

// Two values as a pair of halves and the halves of what is left.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 rest = __ffma2_rn(__half22float2(h), make_float2(-1.0f, -1.0f), make_float2(a, b));  // exact
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The exponent e with max 2^-e in [2^14, 2^15), from the bits of a block's
// largest magnitude, but no lower than `lowest` (which zeros get).  Below
// 2^15 2^lowest a block keeps the absolute step of that size.
__device__ __forceinline__ int block_exponent(uint32_t max_bits, int lowest) {
    return max((int)(max_bits >> 23) - 127 - 14, lowest);
}
// Of queries and keys: the product of the two scales, times log2(e) / sqrt(D), is
// then a normal number, so that it times a masked score of -inf stays -inf (0 * inf
// made NaN of the rows).  What is lost of a score is below 2^-85 of the other factor.
constexpr int kLowestFactor = -60;
// Of values.  A page of zeros (an evicted one) must not stand above a page that has
// values: the weights' reference is the largest score + value exponent, and a page
// of zeros taken as 2^15 pushed all others' weights down into fp16's subnormals
// (values of 1e-3: error 8e-4 instead of 8e-8).
constexpr int kLowestValue = -100;
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // |e| <= 126
// Largest magnitude of three, NaN if one is (one instruction).
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float y;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// One thread of a converged warp.  The tensor-core instructions take their
// operands from uniform registers: in a branch that the compiler knows to hold
// one thread they issue back to back (64 cycles for N = 128, as fast as they
// run); under `lane == 0` each took more than 120.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Moves the executing warpgroup's share of the CTA's registers to R a thread.
template <int R>
__device__ __forceinline__ void set_registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void set_registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace tb
