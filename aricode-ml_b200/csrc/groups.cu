// groups.cu — entry points of the products with group-scaled 4-bit weights (groups.cuh):
// argument checks and launches. Caller's stream, nothing allocated, nothing synchronised.
#include <algorithm>

#include "groups.cuh"
#include "host_checks.cuh"

using namespace b2;

extern "C" {

size_t b2_gemv_i4_groups_workspace(int T, int n) { return 0; }

int b2_gemv_i4_groups(const uint8_t* W, int64_t ld, const void* scale, int64_t lds, int scale_bf16, int group, const float* X,
                      int64_t ldx, const float* bias, float* Y, int64_t ldy, int m, int n, int T, void* workspace,
                      size_t workspace_bytes, void* stream) {
    const char* fn = "b2_gemv_i4_groups";
    if (group != 32 && group != 64 && group != 128) return refuse(fn, "group must be 32, 64 or 128");
    if (m < 0 || n <= 0 || T < 0) return refuse(fn, "m and T must not be negative, n positive");
    if (m == 0 || T == 0) return B2_OK;
    if (!W || !al16(W) || ld % 16 || ld < ((int64_t)n + 1) / 2) return refuse(fn, "W: 16-byte aligned, ld a multiple of 16 that holds a row");
    const int64_t groups = ((int64_t)n + group - 1) / group;
    if (!scale || lds < groups || (reinterpret_cast<uintptr_t>(scale) & (scale_bf16 ? 1 : 3)))
        return refuse(fn, "scale must be set and aligned, lds hold a row");
    if (!X || !Y || !al4(X) || !al4(Y) || !al4(bias) || ldx < n || ldy < m)
        return refuse(fn, "X, Y and bias: 4-byte aligned, row strides that hold a row");
    if (overlap({X, ldx, n}, {Y, ldy, m}, T)) return refuse(fn, "Y overlaps X");
    const size_t need = b2_gemv_i4_groups_workspace(T, n);
    if (need && (!workspace || !al16(workspace) || workspace_bytes < need))
        return refuse(fn, "needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    GroupParams p{};
    p.W = W; p.ld = ld; p.scale = scale; p.lds = lds;
    p.group_log2 = group == 32 ? 5 : group == 64 ? 6 : 7;
    p.x = X; p.ldx = ldx; p.bias = bias; p.y = Y; p.ldy = ldy; p.m = m; p.n = n; p.T = T;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((m + 7) / 8), (unsigned)std::min(T, 65535));
    return status(fn, launch_ex(scale_bf16 ? group_gemv_kernel<true> : group_gemv_kernel<false>, grid, dim3(256), 0, s, true, p));
}

}  // extern "C"
