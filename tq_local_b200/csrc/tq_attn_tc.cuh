// Pieces of the tcgen05 attention kernels: single products with both operands in shared memory, O += P V with the weights in TMEM, TMEM moves of 16
// and 32 columns, arrivals of a warp, and the exponentials of a row.
#pragma once

#include "tq_umma.cuh"

// Instruction descriptor: D = f32, A = B = f16 or bf16, A K-major, N = M = 128; NEGATE: -A.
template <bool BF16, bool TRANSPOSED> __host__ __device__ constexpr uint32_t attn_instr(bool negate = false) {
    return umma_instr<TRANSPOSED>() | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (negate ? 1u << 13 : 0u);
}

// D[128 x 128] (+)= A[128 x 16] * B, both in shared memory
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t instr, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(instr), "r"(accumulate)
        : "memory");
}

// D[128 x 128] (+)= P[128 x 128] * V, P as packed 16-bit pairs in TMEM, V a row-major image (rows are tokens).
__device__ __forceinline__ void attn_values(uint32_t d, uint32_t p, uint32_t v_addr, uint32_t instr, uint32_t accumulate) {
    const uint64_t b = umma_desc<true>(v_addr);
#pragma unroll
    for (uint32_t s = 0; s < 8; ++s) umma_f16(d, p + 8 * s, b + ((s * 16 * 128) >> 4), instr, accumulate | (s > 0));
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {  // tmem_ld_wait before they are used
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {  // tmem_st_wait before anybody reads them
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {  // tmem_st_wait before anybody reads them
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// (the registers are named so that nothing reads them ahead of the wait)
__device__ __forceinline__ void tmem_ld_wait(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ __forceinline__ void mbar_arrive_one(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

// One arrival for a converged warp, after what all of its lanes did before.  (An arrival a lane is 32 operations on one word of shared memory.)
__device__ __forceinline__ void mbar_arrive_warp(uint32_t bar) {
    __syncwarp();
    if (elect_one()) mbar_arrive_one(bar);
}

template <bool BF16> __device__ __forceinline__ uint32_t pack16(float a, float b) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float exp2_hw(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of two numbers without the unit that exp2_hw shares with the whole SM quarter (16 results a clock and SM): the integer nearest to x goes into
// the exponent field, 2 to the rest in [-1/2, 1/2] is the cubic of least relative error (found by Remez exchange; 7.5e-5 = 2^-13.7).
// What is below 2^-125 (-inf too) gives 2^-125: the exponent field does not run over.
__device__ __forceinline__ void exp2_poly(uint64_t x2, float &p, float &q) {
    float a, b;
    f32x2_split(x2, a, b);
    asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(a) : "f"(-125.f));
    asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(b) : "f"(-125.f));
    const uint64_t x = f32x2(a, b), magic = f32x2(12582912.f, 12582912.f);  // 1.5 * 2^23: what is added to it is rounded to an integer
    const uint64_t n = f32x2_add(x, magic);
    const uint64_t f = f32x2_sub(x, f32x2_add(n, f32x2(-12582912.f, -12582912.f)));
    uint64_t y = f32x2_fma(f32x2(0.0551716685f, 0.0551716685f), f, f32x2(0.242611125f, 0.242611125f));
    y = f32x2_fma(y, f, f32x2(0.693260968f, 0.693260968f));
    y = f32x2_fma(y, f, f32x2(0.999928057f, 0.999928057f));
    float na, nb;
    f32x2_split(n, na, nb);
    const float pa = __uint_as_float((__float_as_uint(na) << 23) + 0x3f800000u), pb = __uint_as_float((__float_as_uint(nb) << 23) + 0x3f800000u);
    f32x2_split(f32x2_mul(y, f32x2(pa, pb)), p, q);  // (a product: NaN stays NaN, which adding to its exponent field would not leave)
}
// The running maximum that a row's weights are relative to may lag behind the true one by up to 2^kLag: fp16 weights stay below
// 2^9 and the sums far from overflow, and the accumulator is rescaled a few times a row instead of at every block.
constexpr float kLag = 8.f;
