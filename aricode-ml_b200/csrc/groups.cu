// groups.cu — entry points of the products with group-scaled 4-bit weights (groups.cuh):
// argument checks and launches. Caller's stream, nothing allocated, nothing synchronised.
#include <algorithm>

#include "groups.cuh"
#include "host_checks.cuh"

using namespace b2;

namespace {

constexpr int kVectors = 8;              // of a launch
constexpr size_t kSmem = 227 * 1024;

int fragment_tiles(int T) { return (3 * T + 7) / 8; }          // B columns: three digits of each vector

size_t smem_bytes(int NT, int n) { return NT == 1 ? GroupSmem<1>::bytes(n) : NT == 2 ? GroupSmem<2>::bytes(n) : GroupSmem<3>::bytes(n); }

// Columns of a launch: all of them, or what the shared memory holds of x, in equal parts.
int columns(int NT, int n) {
    int parts = 1, c = n;
    while (smem_bytes(NT, c) > kSmem) {
        ++parts;
        c = ((n + parts - 1) / parts + 511) / 512 * 512;
    }
    return c;
}

// Warps that share a row tile: the fewest pieces (16 rows, 512 columns) one after another.
int share(int m, int n, int sms) {
    const long long tiles = (m + 15) / 16, iters = (n + 511) / 512;
    int best = 1;
    long long least = 0;
    for (int w = 1; w <= kGroupWarps; w *= 2) {
        const long long slots = (long long)sms * (kGroupWarps / w), pieces = (tiles + slots - 1) / slots * ((iters + w - 1) / w);
        if (w == 1 || pieces < least) { best = w; least = pieces; }
    }
    return best;
}

template <int GROUP, int NT, bool BF16>
cudaError_t launch_gemv_groups(const GroupParams& p, int sms, cudaStream_t s) {
    const int smem = (int)smem_bytes(NT, p.n);
    auto k = group_gemv_kernel<GROUP, NT, BF16>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int tiles = (p.m + 15) / 16, slots = kGroupWarps / p.warps_k;
    return launch_ex(k, dim3((unsigned)std::min((tiles + slots - 1) / slots, sms)), dim3(kGroupWarps * 32), smem, s, true, p);
}

template <int GROUP, int NT>
cudaError_t launch_groups(GroupParams p, bool bf16, int sms, cudaStream_t s) {
    if (p.digits) {
        const int words = GroupSmem<NT>::blocks(p.n) * 16;
        cudaError_t e = launch_ex(group_digits_kernel<GROUP, NT>, dim3((unsigned)((words + 255) / 256), (unsigned)p.T), dim3(256), 0, s, true, p);
        if (e != cudaSuccess) return e;
    }
    return bf16 ? launch_gemv_groups<GROUP, NT, true>(p, sms, s) : launch_gemv_groups<GROUP, NT, false>(p, sms, s);
}

template <int GROUP>
cudaError_t launch_groups(const GroupParams& p, int NT, bool bf16, int sms, cudaStream_t s) {
    return NT == 1 ? launch_groups<GROUP, 1>(p, bf16, sms, s) : NT == 2 ? launch_groups<GROUP, 2>(p, bf16, sms, s) : launch_groups<GROUP, 3>(p, bf16, sms, s);
}

}  // namespace

extern "C" {

size_t b2_gemv_i4_groups_workspace(int T, int n) {
    if (T <= 2 || n <= 0) return 0;
    return (size_t)GroupSmem<1>::blocks(n) * fragment_tiles(std::min(T, kVectors)) * (1024 + 32);
}

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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(), unit = scale_bf16 ? 2 : 4;
    for (int t0 = 0; t0 < T; t0 += kVectors) {
        const int NT = fragment_tiles(std::min(T, kVectors)), part = columns(NT, n);
        for (int k0 = 0; k0 < n; k0 += part) {
            GroupParams p{};
            p.W = W + k0 / 2; p.ld = ld;
            p.scale = static_cast<const char*>(scale) + (size_t)(k0 / group) * unit; p.lds = lds;
            p.x = X + (size_t)t0 * ldx + k0; p.ldx = ldx;
            p.bias = k0 ? nullptr : bias;
            p.y = Y + (size_t)t0 * ldy; p.ldy = ldy;
            p.m = m; p.n = std::min(part, n - k0); p.T = std::min(kVectors, T - t0);
            p.add = k0 > 0;
            p.warps_k = share(m, p.n, sms);
            if (T > 2) {
                p.digits = static_cast<uint4*>(workspace);
                p.units = reinterpret_cast<float*>(p.digits + (size_t)GroupSmem<1>::blocks(p.n) * NT * 64);
            }
            const cudaError_t e = group == 32 ? launch_groups<32>(p, NT, scale_bf16, sms, s) : group == 64 ? launch_groups<64>(p, NT, scale_bf16, sms, s)
                                                                                          : launch_groups<128>(p, NT, scale_bf16, sms, s);
            if (e != cudaSuccess) return status(fn, e);
        }
    }
    return B2_OK;
}

}  // extern "C"
