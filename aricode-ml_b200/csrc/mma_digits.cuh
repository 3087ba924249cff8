// mma_digits.cuh — f32 factors as three signed base-256 digits for integer dots on the tensor
// cores: warp-level s8 MMAs, splitting a value, the factor of a set of values. Shared by the
// paged attention and the products with group-scaled 4-bit weights.
#pragma once
#include "b2_common.cuh"

namespace b2 {

// Three digits in [-128, 127] reach 2^23 - 1 - 0x8080 = 8355711; a little below it,
// so that the roundings of factor and product stay inside
constexpr int kDigitMax = 8355700;

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the first of a chain: from zero, so that nothing has to be cleared
__device__ __forceinline__ void mma_s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// the same from a value that all four sums start with
__device__ __forceinline__ void mma_s8_from(int (&c)[4], uint32_t from, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(from));
}

// rint(x f) + 0x8080 for |x f| <= kDigitMax, in the low 24 bits
__device__ __forceinline__ uint32_t digit_bits(float x, float f) { return (uint32_t)__float2int_rn(x * f) + 0x8080u; }
// the same for x >= 0 in one operation: the f32 addition rounds x f to an integer
constexpr float kDigitBase = 8388608.0f + (float)0x8080;
__device__ __forceinline__ uint32_t digit_bits_pos(float x, float f) { return __float_as_uint(ffma(x, f, kDigitBase)); }

// digits of four integers given as digit_bits: word e of d holds digit e of each in its bytes
__device__ __forceinline__ void digits4(uint32_t y0, uint32_t y1, uint32_t y2, uint32_t y3, uint32_t (&d)[3]) {
    const uint32_t l = __byte_perm(y0, y1, 0x5140), m = __byte_perm(y2, y3, 0x5140);
    d[0] = __byte_perm(l, m, 0x5410) ^ 0x80808080u;
    d[1] = __byte_perm(l, m, 0x7632) ^ 0x80808080u;
    d[2] = __byte_perm(__byte_perm(y0, y1, 0x0062), __byte_perm(y2, y3, 0x0062), 0x5410);
}

// the factor that takes values up to `top` (>= 0) to integers up to kDigitMax; tiny
// tops (below 1e-31) keep fewer bits, 0 gives 0, NaN and infinity NaN
__device__ __forceinline__ float digit_factor(float top) {
    if (!(top < __int_as_float(0x7f800000))) return __int_as_float(0x7fffffff);
    return top > 0.0f ? fminf(fdiv((float)kDigitMax, top), 0x1p126f) : 0.0f;
}

}  // namespace b2
