// groups.cuh — products with 4-bit weights that have a scale for each row and group of
// columns (sm_100a).
#pragma once
#include "kernels.cuh"

namespace b2 {

struct GroupParams {
    const uint8_t* W;        // [m][ld] packed codes, the even column in the low half
    long long ld;
    const void* scale;       // [m][lds] f32 or bf16
    long long lds;
    int group_log2;
    const float* x;          // [T][ldx]
    long long ldx;
    const float* bias;       // [m] or nullptr
    float* y;                // [T][ldy]
    long long ldy;
    int m, n, T;
};

template <bool BF16>
__device__ __forceinline__ float group_scale(const void* scale, size_t i) {
    if constexpr (BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(scale)[i] << 16);
    else return static_cast<const float*>(scale)[i];
}

// One warp a row and vector.
template <bool BF16>
__global__ void __launch_bounds__(256) group_gemv_kernel(const __grid_constant__ GroupParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= p.m) return;
    for (int t = blockIdx.y; t < p.T; t += gridDim.y) {
        const float* x = p.x + (size_t)t * p.ldx;
        float y = 0.0f, off = 0.0f;                            // off: NaN where x is not finite
        for (int g = 0; g << p.group_log2 < p.n; ++g) {
            const int end = min((g + 1) << p.group_log2, p.n);
            float a = 0.0f;
            for (int k = (g << p.group_log2) + lane; k < end; k += 32) {
                const int b = p.W[(size_t)row * p.ld + (k >> 1)] >> (4 * (k & 1)) & 15;
                a = ffma((float)((b ^ 8) - 8), x[k], a);
                off = ffma(x[k], 0.0f, off);
            }
            y = ffma(a, group_scale<BF16>(p.scale, (size_t)row * p.lds + g), y);
        }
        y = butterfly32(y + off);
        if (lane == 0) p.y[(size_t)t * p.ldy + row] = p.bias ? fadd(y, p.bias[row]) : y;
    }
}

}  // namespace b2
