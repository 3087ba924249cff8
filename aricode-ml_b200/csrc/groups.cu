// groups.cu — entry points of the products with group-scaled 4-bit weights (groups.cuh):
// argument checks and launches. Caller's stream, nothing allocated, nothing synchronised.
#include <algorithm>

#include "groups.cuh"
#include "host_checks.cuh"
#include "tensor_map.cuh"

using namespace b2;

namespace {

// Up to 8 vectors (three fragments of their digits) the first kind of kernel, else the second. 8 vectors by the first and
// the second, us in a captured graph: 5632 x 2048, groups of 32 12 and 19; 4096 x 4096 12 and 18; 32000 x 4096 39 and 55;
// 4096 x 11008, whose columns are two launches of the first then, 27 and 27. 3 vectors: 12 and 16, 12 and 16, 33 and 55, 21
// and 25. (The first for more than 8, with more fragments, is not written.)
constexpr int kVectors = 8;
constexpr int kGemmVectors = 64;         // of a launch of the second kind
constexpr size_t kSmem = 227 * 1024;
constexpr int kMost = 0x7fff0000;        // of m, n and T: what goes past them by a tile or a round of tiles stays in 32 bits

int fragment_tiles(int T) { return (3 * T + 7) / 8; }          // B columns: three digits of each vector

size_t smem_bytes(int NT, int n) { return NT == 1 ? GroupSmem<1>::bytes(n) : NT == 2 ? GroupSmem<2>::bytes(n) : GroupSmem<3>::bytes(n); }

// Columns of a launch: all of them, or what the shared memory holds of x, in equal parts.
int columns(int NT, int n) {
    int parts = 1, c = n;
    while (smem_bytes(NT, c) > kSmem) {
        ++parts;
        c = (int)(((((long long)n + parts - 1) / parts + 511) / 512) * 512);
    }
    return c;
}

// Warps that share a row tile: the fewest pieces (16 rows, 512 columns) one after another, a meeting for a quarter of
// one (32000 x 4096: 7 pieces and as many meetings 24.0 us, 8 and none 22.2).
int share(int m, int n, int sms) {
    const long long tiles = (m + 15) / 16, iters = (n + 511) / 512;
    int best = 1;
    long long least = 0;
    for (int w = 1; w <= kGroupWarps; w *= 2) {
        const long long slots = (long long)sms * (kGroupWarps / w), cost = (tiles + slots - 1) / slots * (4 * ((iters + w - 1) / w) + (w > 1));
        if (w == 1 || cost < least) { best = w; least = cost; }
    }
    return best;
}

template <int GROUP, int NT, bool BF16>
cudaError_t launch_gemv_groups(const GroupParams& p, int sms, cudaStream_t s) {
    const int smem = (int)smem_bytes(NT, p.n);
    auto k = group_gemv_kernel<GROUP, NT, BF16>;
    cudaError_t e = allow_smem<group_gemv_kernel<GROUP, NT, BF16>>((int)kSmem);      // (whatever other threads' calls need)
    if (e != cudaSuccess) return e;
    return launch_ex(k, dim3((unsigned)std::min((p.m + 15) / 16, sms)), dim3(kGroupWarps * 32), smem, s, true, p);
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

// images and units of a block of 128 columns, parts of row tiles
size_t gemm_bytes(int NT, int n, int sms) { return (size_t)GroupSmem<1>::blocks(n) * NT * (512 + 4) + (size_t)sms * 2 * NT * 128 * sizeof(float); }

int gemm_vectors(int T) { return T <= 16 ? 16 : T <= 32 ? 32 : kGemmVectors; }

template <int GROUP, int NT, bool BF16>
cudaError_t launch_gemm(const GemmParams& p, int sms, cudaStream_t s) {
    auto k = group_gemm_kernel<GROUP, NT, BF16>;
    cudaError_t e = allow_smem<group_gemm_kernel<GROUP, NT, BF16>>(GemmShape<GROUP, NT>::Alloc);
    if (e != cudaSuccess) return e;
    const int tiles = (p.m + 127) / 128, steps = tiles * GroupSmem<1>::blocks(p.n), ctas = std::min(steps, sms);
    e = launch_ex(k, dim3((unsigned)ctas), dim3(kGemmThreads), GemmShape<GROUP, NT>::Alloc, s, true, p);
    if (e != cudaSuccess || ctas == tiles) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles, (unsigned)p.T);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1] = {pdl_attr(true)};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, group_add_kernel<NT>, p, ctas);
}

template <int NT>
cudaError_t launch_gemm(const GroupParams& g, int group, bool bf16, int sms, cudaStream_t s) {
    GemmParams p{};
    EncodeTiled enc = tensor_map_encoder();
    if (!enc) return cudaErrorNotSupported;
    // (a row's own bytes and no more: rows may be columns of a wider matrix, and the last one end with it)
    const cuuint64_t dims[2] = {((cuuint64_t)g.n + 1) / 2, (cuuint64_t)g.m}, strides[1] = {(cuuint64_t)g.ld};
    const cuuint32_t box[2] = {64, 128}, step[2] = {1, 1};
    if (enc(&p.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(g.W), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    p.scale = g.scale; p.lds = g.lds; p.bias = g.bias; p.y = g.y; p.ldy = g.ldy; p.m = g.m; p.n = g.n; p.T = g.T;
    p.images = reinterpret_cast<const unsigned char*>(g.digits); p.units = g.units;
    p.part = g.units + (size_t)GroupSmem<1>::blocks(g.n) * NT;
    const int words = GroupSmem<1>::blocks(g.n) * 16;
    cudaError_t e = launch_ex(group_images_kernel<NT>, dim3((unsigned)((words + 255) / 256), (unsigned)g.T), dim3(256), 0, s, true, g);
    if (e != cudaSuccess) return e;
#define B2_CALL(G) (bf16 ? launch_gemm<G, NT, true>(p, sms, s) : launch_gemm<G, NT, false>(p, sms, s))
    return group == 32 ? B2_CALL(32) : group == 64 ? B2_CALL(64) : B2_CALL(128);
#undef B2_CALL
}

}  // namespace

extern "C" {

size_t b2_gemv_i4_groups_workspace(int T, int n) {
    if (T <= 2 || n <= 0 || T > kMost || n > kMost) return 0;
    if (T > kVectors) return gemm_bytes(gemm_vectors(T), n, sm_count());
    return (size_t)GroupSmem<1>::blocks(n) * fragment_tiles(T) * (1024 + 32);
}

int b2_gemv_i4_groups(const uint8_t* W, int64_t ld, const void* scale, int64_t lds, int scale_bf16, int group, const float* X,
                      int64_t ldx, const float* bias, float* Y, int64_t ldy, int m, int n, int T, void* workspace,
                      size_t workspace_bytes, void* stream) {
    const char* fn = "b2_gemv_i4_groups";
    if (group != 32 && group != 64 && group != 128) return refuse(fn, "group must be 32, 64 or 128");
    if (m < 0 || n <= 0 || T < 0) return refuse(fn, "m and T must not be negative, n positive");
    if (m > kMost || n > kMost || T > kMost) return refuse(fn, "m, n and T: at most 2^31 - 2^16");
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
    const Bytes read[] = {rows_bytes(W, ld, ((int64_t)n + 1) / 2, m, 1), rows_bytes(scale, lds, groups, m, scale_bf16 ? 2 : 4),
                          {bias, 4ll * m}, rows_bytes(X, ldx, n, T, 4)};
    const Bytes y = rows_bytes(Y, ldy, m, T, 4), ws = {workspace, (int64_t)need};
    if (touch(y, {read[0], read[1], read[2], ws})) return refuse(fn, "Y overlaps W, scale, bias or the workspace");
    if (touch(ws, read)) return refuse(fn, "the workspace overlaps an input");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(), unit = scale_bf16 ? 2 : 4;
    if (T > kVectors) {
        for (int t0 = 0; t0 < T; t0 += kGemmVectors) {
            GroupParams p{};
            p.W = W; p.ld = ld; p.scale = scale; p.lds = lds; p.bias = bias;
            p.x = X + (size_t)t0 * ldx; p.ldx = ldx; p.y = Y + (size_t)t0 * ldy; p.ldy = ldy;
            p.m = m; p.n = n; p.T = std::min(kGemmVectors, T - t0);
            const int NT = gemm_vectors(T);
            p.digits = static_cast<uint4*>(workspace);
            p.units = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + (size_t)GroupSmem<1>::blocks(n) * NT * 512);
            const cudaError_t e = NT == 16 ? launch_gemm<16>(p, group, scale_bf16, sms, s) : NT == 32 ? launch_gemm<32>(p, group, scale_bf16, sms, s)
                                                                                                   : launch_gemm<64>(p, group, scale_bf16, sms, s);
            if (e != cudaSuccess) return status(fn, e);
        }
        return B2_OK;
    }
    const int NT = fragment_tiles(T), part = columns(NT, n);
    for (int k0 = 0; k0 < n; k0 += part) {
        GroupParams p{};
        p.W = W + k0 / 2; p.ld = ld;
        p.scale = static_cast<const char*>(scale) + (size_t)(k0 / group) * unit; p.lds = lds;
        p.x = X + k0; p.ldx = ldx;
        p.bias = k0 ? nullptr : bias;
        p.y = Y; p.ldy = ldy;
        p.m = m; p.n = std::min(part, n - k0); p.T = T;
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
    return B2_OK;
}

}  // extern "C"
