// groups.cuh — products with 4-bit weights that have a scale for each row and group of
// columns (sm_100a).
//
//   y[t][j] = sum_g s[j][g] sum_{k in g} c[j][k] x[t][k]
//
// The codes are exact small integers, so a group's sum runs as an integer dot on the tensor
// cores, with x split into three signed base-256 digits: X = rint(x f) = d2 65536 + d1 256
// + d0, f from the largest of each 128 neighbours (a channel that stands out costs its
// neighbours alone). The digit sums are exact in int32; each is scaled by s and 1 / f into a
// f32 sum of its own, and the three are joined at the end.
#pragma once
#include "mma_digits.cuh"
#include "paged_rows.cuh"

namespace b2 {

struct GroupParams {
    const uint8_t* W;        // [m][ld] packed codes, the even column in the low half
    long long ld;
    const void* scale;       // [m][lds] f32 or bf16
    long long lds;
    const float* x;          // [T][ldx]
    long long ldx;
    const float* bias;       // [m] or nullptr
    float* y;                // [T][ldy]
    long long ldy;
    int m, n, T;
    int add;                 // columns before these are in y already
    int warps_k;             // warps that share a row tile's columns: 1, 2, 4, 8 or 16
    uint4* digits;           // [blocks][NT][2][32]: x as B fragments (nullptr: made by each CTA)
    float* units;            // [blocks][8 NT]: what an integer unit of a column stands for
};

template <bool BF16>
__device__ __forceinline__ float group_scale(const void* scale, size_t i) {
    if constexpr (BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(scale)[i] << 16);
    else return static_cast<const float*>(scale)[i];
}

// A block of 128 columns is four MMAs of 32. In the rows of W lane t of a quad loads the 16
// bytes (32 columns) number t; the words change lanes so that an MMA's columns lie in one
// group: MMA u takes of lane t
//   group 128: word u of its own 16 bytes
//   group  64: (u < 2: columns 0 .. 63) word u of lanes 0, 1, word u + 2 of the same bytes in lanes 2, 3
//   group  32: word t of the 16 bytes number u
// so x's columns 8 w .. 8 w + 7 of a block (word w) stand at (MMA, lane) = place(w).
template <int GROUP>
__device__ __forceinline__ int2 group_place(int w) {
    const int chunk = w >> 2, i = w & 3;
    if constexpr (GROUP == 128) return make_int2(i, chunk);
    if constexpr (GROUP == 32) return make_int2(chunk, i);
    return make_int2((chunk & 2) + (i & 1), (chunk & 1) + (i & 2));
}

// words of MMAs 0 .. 3 from the lane's 16 bytes
template <int GROUP>
__device__ __forceinline__ void group_words(const uint4& v, uint32_t (&w)[4], int t) {
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    if constexpr (GROUP <= 64) {                               // between lanes t and t ^ 2: words 2, 3 against 0, 1
        const bool up = t & 2;
        const uint32_t a = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[2], 2), b = __shfl_xor_sync(0xffffffffu, up ? w[1] : w[3], 2);
        if (up) { w[0] = a; w[1] = b; }
        else { w[2] = a; w[3] = b; }
    }
    if constexpr (GROUP == 32) {                               // between t and t ^ 1: the odd word against the even one
        const bool up = t & 1;
        const uint32_t a = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[1], 1), b = __shfl_xor_sync(0xffffffffu, up ? w[2] : w[3], 1);
        if (up) { w[0] = a; w[2] = b; }
        else { w[1] = a; w[3] = b; }
    }
}

// One word of a vector (columns 8 w .. + 7 of block kb) as digits, by 16 neighbouring lanes for
// a block: fragments to `frag` ([NT][2][32] uint4 of this block), units to `unit` ([8 NT]).
// Rows of x may start anywhere. All lanes of the warp take part; `live`: t is a vector.
template <int GROUP>
__device__ __forceinline__ void group_digits(const GroupParams& p, int t, int kb, int w, bool live, uint4* frag, float* unit) {
    float x[8], top = 0.0f;
    const int k0 = kb * 128 + 8 * w;
    const float* src = p.x + (size_t)t * p.ldx + k0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = live && k0 + i < p.n ? src[i] : 0.0f;
        bad |= x[i] != x[i];
        top = fmaxf(top, fabsf(x[i]));
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) return;
    const float f = digit_factor(top);
    uint32_t even[3], odd[3];
    digits4(digit_bits(x[0], f), digit_bits(x[2], f), digit_bits(x[4], f), digit_bits(x[6], f), even);
    digits4(digit_bits(x[1], f), digit_bits(x[3], f), digit_bits(x[5], f), digit_bits(x[7], f), odd);
    const int2 at = group_place<GROUP>(w);
#pragma unroll
    for (int e = 0; e < 3; ++e) {
        const int col = 3 * t + e;
        uint2* q = reinterpret_cast<uint2*>(frag + ((col >> 3) * 2 + (at.x >> 1)) * 32 + (col & 7) * 4 + at.y);
        q[at.x & 1] = make_uint2(even[e], odd[e]);
        // the codes enter as 16 c; digit e counts 256^e, which the end multiplies in
        if (w == 0) unit[col] = f > 0.0f ? fdiv(0.0625f, f) : f;
    }
}

template <int GROUP, int NT>
__global__ void __launch_bounds__(256) group_digits_kernel(const __grid_constant__ GroupParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int word = blockIdx.x * 256 + threadIdx.x, kb = word >> 4, t = blockIdx.y;
    const bool live = kb * 128 < p.n;
    group_digits<GROUP>(p, t, live ? kb : 0, word & 15, live, p.digits + (size_t)kb * NT * 64, p.units + (size_t)kb * NT * 8);
}

// y for up to 8 NT / 3 vectors. Bound by memory: a CTA a SM goes through the row tiles of 16;
// warps_k warps share a tile's columns (512 at a time each, the next 512 requested before these are
// used, across tiles too) and meet in shared memory. x's digits are B fragments in shared
// memory, made by the CTA itself for one or two vectors, else by a launch before.
constexpr int kGroupWarps = 16;

template <int NT>
struct GroupSmem {
    static constexpr int RedFloats = kGroupWarps * 16 * 8 * NT;    // a warp's sums [16 rows][8 NT]
    static int blocks(int n) { return (n + 127) / 128; }
    static size_t bytes(int n) { return (size_t)blocks(n) * NT * (1024 + 32) + 2 * RedFloats * sizeof(float); }
};

template <int GROUP, int NT, bool BF16>
__global__ void __launch_bounds__(kGroupWarps * 32) group_gemv_kernel(const __grid_constant__ GroupParams p) {
    extern __shared__ __align__(16) unsigned char gg_raw[];
    constexpr int GB = 128 / GROUP;                            // groups in a block
    constexpr uint32_t kMagic = 0x4b400000u;                   // 1.5 2^23: its sum with |i| < 2^22, read as a float
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int blocks = (p.n + 127) >> 7, iters = (p.n + 511) >> 9, chunks = (p.n + 31) >> 5, groups = (p.n + GROUP - 1) / GROUP;
    const int tiles = (p.m + 15) >> 4, slots = kGroupWarps / p.warps_k, slot = warp / p.warps_k, wk = warp % p.warps_k;
    uint4* frag = reinterpret_cast<uint4*>(gg_raw);
    float* unit = reinterpret_cast<float*>(frag + (size_t)blocks * NT * 64);
    float* red = unit + (size_t)blocks * NT * 8;
    pdl_launch_dependents();
    pdl_wait();

    // this warp's pieces: (tile, 512 columns)
    int tile = blockIdx.x * slots + slot, it = wk;
    uint4 w0[4], w1[4];                                        // rows g and g + 8 of the tile, blocks 4 it ..
    float s0[GB], s1[GB];                                      // their scales: lane t has number 4 i + t of the piece
    auto load = [&](int tile, int it) {
        const bool there = tile < tiles && it < iters;
        const int r0 = min(tile * 16 + g, p.m - 1), r1 = min(tile * 16 + g + 8, p.m - 1);
        const uint8_t* a = p.W + (size_t)r0 * p.ld + 64ll * 4 * it + 16 * t;
        const uint8_t* b = p.W + (size_t)r1 * p.ld + 64ll * 4 * it + 16 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = there && 16 * it + 4 * i + t < chunks;
            w0[i] = in ? load16(a + 64 * i) : make_uint4(0u, 0u, 0u, 0u);
            w1[i] = in ? load16(b + 64 * i) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < GB; ++i) {
            const int gi = 4 * GB * it + 4 * i + t;
            const bool in = there && gi < groups;
            s0[i] = in ? group_scale<BF16>(p.scale, (size_t)r0 * p.lds + gi) : 0.0f;
            s1[i] = in ? group_scale<BF16>(p.scale, (size_t)r1 * p.lds + gi) : 0.0f;
        }
    };
    load(tile, it);
    if (p.digits) {
        for (int i = tid; i < blocks * NT * 64; i += kGroupWarps * 32) frag[i] = p.digits[i];
        for (int i = tid; i < blocks * NT * 8; i += kGroupWarps * 32) unit[i] = p.units[i];
    } else {
        for (int word = tid; word < (blocks + 1) / 2 * 32 * p.T; word += kGroupWarps * 32) {       // whole warps: two blocks of a vector
            const int half = word >> 4, v = half / (2 * ((blocks + 1) / 2)), kb = half % (2 * ((blocks + 1) / 2));
            group_digits<GROUP>(p, v, kb, word & 15, kb < blocks, frag + (size_t)kb * NT * 64, unit + (size_t)kb * NT * 8);
        }
    }
    __syncthreads();

    float acc[NT][4];
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[y][i] = 0.0f;
    // (every warp of a slot runs the same number of pieces a tile, so that they meet)
    const int per_tile = (iters + p.warps_k - 1) / p.warps_k;
    for (int step = 0, buf = 0; tile < tiles; ) {
        const int kb0 = 4 * it;
        const bool mine = it < iters;
        uint32_t a[4][2][4];                                   // [block][row half][MMA]
        float sc0[GB], sc1[GB];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            group_words<GROUP>(w0[i], a[i][0], t);
            group_words<GROUP>(w1[i], a[i][1], t);
        }
#pragma unroll
        for (int i = 0; i < GB; ++i) { sc0[i] = s0[i]; sc1[i] = s1[i]; }
        const int cur = tile;
        const bool last = ++step == per_tile;
        it += p.warps_k;
        if (last) {
            step = 0;
            it = wk;
            tile += gridDim.x * slots;
        }
        load(tile, it);
        if (mine) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int kb = kb0 + i;
                if (kb >= blocks) break;
                const uint4* fb = frag + (size_t)kb * NT * 64 + lane;
#pragma unroll
                for (int y = 0; y < NT; ++y) {
                    const uint4 b01 = fb[y * 64], b23 = fb[y * 64 + 32];
                    const float2 un = *reinterpret_cast<const float2*>(unit + (kb * NT + y) * 8 + 2 * t);
                    const f32x2 u2 = pack2(un.x, un.y);
                    int c[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t x = a[i][0][u], z = a[i][1][u];
                        const uint32_t e0 = (x << 4) & 0xf0f0f0f0u, e1 = (z << 4) & 0xf0f0f0f0u, o0 = x & 0xf0f0f0f0u, o1 = z & 0xf0f0f0f0u;
                        const uint32_t b0 = u == 0 ? b01.x : u == 1 ? b01.z : u == 2 ? b23.x : b23.z;
                        const uint32_t b1 = u == 0 ? b01.y : u == 1 ? b01.w : u == 2 ? b23.y : b23.w;
                        if (u % (4 / GB) == 0) mma_s8_from(c, kMagic, e0, e1, o0, o1, b0, b1);
                        else mma_s8(c, e0, e1, o0, o1, b0, b1);
                        if ((u + 1) % (4 / GB) == 0) {         // the group is complete
                            const int gi = i * GB + u / (4 / GB);      // of the piece; lane gi % 4 has its scales
                            const float r0 = __shfl_sync(0xffffffffu, sc0[gi >> 2], (lane & 28) + (gi & 3));
                            const float r1 = __shfl_sync(0xffffffffu, sc1[gi >> 2], (lane & 28) + (gi & 3));
                            const f32x2 off = pack2(-12582912.0f, -12582912.0f);
                            const f32x2 v0 = add2(pack2(__int_as_float(c[0]), __int_as_float(c[1])), off);
                            const f32x2 v1 = add2(pack2(__int_as_float(c[2]), __int_as_float(c[3])), off);
                            const float2 y0 = unpack2(fma2(v0, mul2(pack2(r0, r0), u2), pack2(acc[y][0], acc[y][1])));
                            const float2 y1 = unpack2(fma2(v1, mul2(pack2(r1, r1), u2), pack2(acc[y][2], acc[y][3])));
                            acc[y][0] = y0.x; acc[y][1] = y0.y; acc[y][2] = y1.x; acc[y][3] = y1.y;
                        }
                    }
                }
            }
        }
        if (!last) continue;
        // the tile's sums meet: [row][column] of each warp
        float* rw = red + buf * GroupSmem<NT>::RedFloats;
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            float* q = rw + (warp * 16 + g) * 8 * NT + 8 * y + 2 * t;
            *reinterpret_cast<float2*>(q) = make_float2(acc[y][0], acc[y][1]);
            *reinterpret_cast<float2*>(q + 8 * 8 * NT) = make_float2(acc[y][2], acc[y][3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[y][i] = 0.0f;
        }
        if (p.warps_k > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(p.warps_k * 32) : "memory");
        else __syncwarp();
        for (int i = wk * 32 + lane; i < 16 * p.T; i += p.warps_k * 32) {
            const int row = cur * 16 + i % 16, v = i / 16;
            if (row >= p.m) continue;
            const float* q = rw + (slot * p.warps_k * 16 + i % 16) * 8 * NT + 3 * v;
            float d0 = 0.0f, d1 = 0.0f, d2 = 0.0f;
            for (int w = 0; w < p.warps_k; ++w, q += 16 * 8 * NT) { d0 += q[0]; d1 += q[1]; d2 += q[2]; }
            float y = ffma(d2, 65536.0f, ffma(d1, 256.0f, d0)), *out = p.y + (size_t)v * p.ldy + row;
            if (p.bias) y = fadd(y, p.bias[row]);
            *out = p.add ? fadd(*out, y) : y;
        }
        buf ^= 1;
    }
}

}  // namespace b2
