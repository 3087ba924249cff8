// f16_pairs.cuh — f32 factors as two f16 each for products on the tensor cores, after a power
// of two has brought the largest of a set into range: 22 bits of an element. Shared by the
// tree attention and the products with group-scaled 4-bit weights.
#pragma once
#include <cuda_fp16.h>

#include "b2_common.cuh"

namespace b2 {

// two values as two f16 each: hi the nearest, lo what is left
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

constexpr int kRowBits = 13;                       // of rows of f32 factors: the largest at [2^13, 2^14)

// the power of two that brings `top` (finite, >= 0) to [2^bits, 2^(bits + 1)), and its reciprocal;
// tiny ones are brought as far as 2^126 does
__device__ __forceinline__ void f16_factor(float top, int bits, float& f, float& unit) {
    const int e = min(max(bits + 254 - (int)(__float_as_uint(top) >> 23), 1), 253);
    f = __int_as_float(e << 23);
    unit = __int_as_float((254 - e) << 23);
}

}  // namespace b2
