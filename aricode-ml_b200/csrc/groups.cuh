// groups.cuh — products with 4-bit weights that have a scale for each row and group of
// columns (sm_100a).
//
//   y[t][j] = sum_g s[j][g] sum_{k in g} c[j][k] x[t][k]
//
// The codes are exact small integers, so a group's sum runs as an integer dot on the tensor
// cores, with x split into three signed base-256 digits: X = rint(x f) = d2 65536 + d1 256
// + d0, f from the largest of each 128 neighbours (a channel that stands out costs its
// neighbours alone). The digit sums are exact in int32; each is scaled by 256^e / f and s into a
// f32 sum of its own, and the three are joined at the end.
#pragma once
#include "f16_pairs.cuh"
#include "mma_digits.cuh"
#include "paged_rows.cuh"
#include "umma.cuh"

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

// Sums are held over this: of x's largest value a group's sum is up to 8 x 128 times that, which its scale may bring back.
// (Their smallest normal number is 2^-126 times this then.)
constexpr float kGroupRoom = 1024.0f;

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
        // the codes enter as 16 c; digit e counts 256^e; all over kGroupRoom
        if (w == 0) unit[col] = f > 0.0f ? fdiv((e == 0 ? 0.0625f : e == 1 ? 16.0f : 4096.0f) / kGroupRoom, f) : f;
    }
}

template <int GROUP, int NT>
__global__ void __launch_bounds__(256) group_digits_kernel(const __grid_constant__ GroupParams p) {
    pdl_wait();
    pdl_launch_dependents();                                   // (not before: what the products read besides is ready then)
    const int word = blockIdx.x * 256 + threadIdx.x, kb = word >> 4, t = blockIdx.y;
    const bool live = kb * 128 < p.n;
    group_digits<GROUP>(p, t, live ? kb : 0, word & 15, live, p.digits + (size_t)kb * NT * 64, p.units + (size_t)kb * NT * 8);
}

// y for up to 8 NT / 3 vectors. Bound by memory: a CTA a SM goes through the row tiles of 16;
// warps_k warps share a tile's columns (512 at a time each, the next 512 requested before these are
// used, across tiles too) and meet in shared memory. x's digits are B fragments in shared
// memory, made by the CTA itself for one or two vectors, else by a launch before.
// 32000 x 4096, one vector: 21.3 us (10.7 at 6.56 TB/s); 22.2 with 16 neighbouring tiles a CTA, which leaves 23 SMs none.
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
    if (!p.digits) pdl_wait();                                 // (else behind the first weights, which are ready)

    // this warp's pieces: (tile, 512 columns)
    int tile = slot * gridDim.x + blockIdx.x, it = wk;         // (tiles over all SMs before a second one on any)
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
        pdl_wait();
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
                            // (unit x scale first could be too small for f32 where their product with the sum is not)
                            const float2 y0 = unpack2(fma2(mul2(v0, u2), pack2(r0, r0), pack2(acc[y][0], acc[y][1])));
                            const float2 y1 = unpack2(fma2(mul2(v1, u2), pack2(r1, r1), pack2(acc[y][2], acc[y][3])));
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
            float y = kGroupRoom * fadd(d2, fadd(d1, d0)), *out = p.y + (size_t)v * p.ldy + row;
            if (p.bias) y = fadd(y, p.bias[row]);
            *out = p.add ? fadd(*out, y) : y;
        }
        buf ^= 1;
    }
}

// ---- more vectors: the 5th-generation tensor cores. Per 128 columns, D [row][vector] = W X^T in
// f16 with W's codes (exact) as 128 x 128 tiles and x as two f16 each (f16_pairs.cuh), lo and then
// hi into the same sums (side by side, as 2 NT columns, the MMAs took two thirds of the time, but
// what is bound is reading the sums); a D for each group, so that its scale and x's unit (for each 128 columns of a
// vector) come in f32 behind it. Sums in the tensor cores are a group long.
// A CTA a SM has an equal share of the (128 rows, 128 columns) steps in order: parts of row
// tiles and whole ones; parts' sums go to the workspace and are added in order of columns.
// Warps 0 .. 7: sums to f32: warp w has TMEM lanes (rows) 32 (w % 4) .. + 31 and half w / 4 of the vectors.
// Warps 8 .. 15: codes to f16 operands. Warps 16, 17: copies (packed rows by TMA; x's images and units
// by bulk copies, behind the launch that makes them: one warp for all was what a step waited for). Warp
// 18: issues the MMAs. Every wait is bounded. 4096 x 11008, 64 vectors: 27 us (weights alone 4); 5632 x 2048, 13: 14.
constexpr int kGemmSumWarps = 8, kGemmConvWarps = 8;
constexpr int kTeam = kGemmConvWarps / 2 * 32;                 // threads that turn a step's codes
constexpr int kGemmThreads = (kGemmSumWarps + kGemmConvWarps + 3) * 32;

template <int GROUP, int NT>
struct GemmShape {
    static constexpr int Image = NT * 512;                     // x of 128 columns: [half][hi, lo of NT vectors][64 f16], swizzled
    static constexpr int Units = NT * 4;                       // and what a unit of them is, by vector
    static constexpr int Tile = 128 * 256;                     // codes as f16: [half][row][64 f16], swizzled
    static constexpr int Packed = 128 * 64;                    // codes as they come: [row][64 bytes]
    static constexpr int SX = NT == 64 ? 3 : 4, SW = NT == 64 ? 6 : 8, SA = 2;
    static constexpr int GS = 128 / GROUP;                     // groups of a step
    static constexpr int DB = 8;                               // sums in TMEM
    static constexpr int A = 0;
    static constexpr int X = A + SA * Tile;
    static constexpr int W = X + SX * Image;
    static constexpr int U = W + SW * Packed;
    static constexpr int Bars = U + SX * Units;
    static constexpr int NBars = 2 * SA + 2 * SX + 2 * SW + 2 * DB + 1;
    static constexpr int Alloc = Bars + NBars * 8 + 16 + 1024;
    static constexpr int TmemCols = DB * NT;
    static_assert(Alloc <= 227 * 1024, "");
};

struct GemmParams {
    CUtensorMap W;           // [m][ld] bytes
    const void* scale;
    long long lds;
    const unsigned char* images;   // [blocks][GemmShape::Image]
    const float* units;            // [blocks][NT]
    const float* bias;
    float* y;
    long long ldy;
    int m, n, T;
    float* part;             // [CTA][2][NT][128]: its first and its last part of a row tile
};

// The first of a CTA's steps (of blocks steps for each row tile), and the CTA that has a step.
__device__ __forceinline__ int gemm_first(int steps, int ctas, int cta) { return cta * (steps / ctas) + min(cta, steps % ctas); }
__device__ __forceinline__ int gemm_cta(int steps, int ctas, int at) {
    const int each = steps / ctas, more = steps % ctas, turn = more * (each + 1);
    return at < turn ? at / (each + 1) : more + (at - turn) / each;
}

// x as images: words of 8 columns, 16 lanes for a block of 128; in each word the columns stand as
// the codes come out of it: 0 4 1 5 2 6 3 7
template <int NT>
__global__ void __launch_bounds__(256) group_images_kernel(const __grid_constant__ GroupParams p) {
    pdl_wait();
    pdl_launch_dependents();                                   // (not before: what the products read besides is ready then)
    const int word = blockIdx.x * 256 + threadIdx.x, kb = word >> 4, w = word & 15, t = blockIdx.y;
    const bool live = kb * 128 < p.n;
    const int k0 = kb * 128 + 8 * w;
    const float* src = p.x + (size_t)t * p.ldx + k0;
    float x[8], top = 0.0f;
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
    float f, unit;
    f16_factor(top, kRowBits, f, unit);
    const bool fine = top < INFINITY;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_f16(fine ? x[i] * f : 0.0f, fine ? x[i + 4] * f : 0.0f, hi[i], lo[i]);
    if (w == 0) p.units[(size_t)kb * NT + t] = fine ? unit * (1.0f / kGroupRoom) : __int_as_float(0x7fffffff);
    unsigned char* image = reinterpret_cast<unsigned char*>(p.digits) + (size_t)kb * (NT * 512) + (w >> 3) * (NT * 256);
    *reinterpret_cast<uint4*>(image + t * 128 + (((w & 7) ^ (t & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(image + (NT + t) * 128 + (((w & 7) ^ (t & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

template <int GROUP, int NT, bool BF16>
__global__ void __launch_bounds__(kGemmThreads, 1) group_gemm_kernel(const __grid_constant__ GemmParams p) {
    using Sh = GemmShape<GROUP, NT>;
    constexpr int GS = Sh::GS, DB = Sh::DB;
    extern __shared__ unsigned char gm_raw[];
    unsigned char* sm = gm_raw + ((1024u - (smem_u32(gm_raw) & 1023u)) & 1023u);
    uint64_t* wfull = reinterpret_cast<uint64_t*>(sm + Sh::Bars);      // [SW] packed codes have come
    uint64_t* wempty = wfull + Sh::SW;
    uint64_t* xfull = wempty + Sh::SW;                                 // [SX] an image and its units
    uint64_t* xempty = xfull + Sh::SX;
    uint64_t* afull = xempty + Sh::SX;                                 // [SA] codes as f16
    uint64_t* aempty = afull + Sh::SA;
    uint64_t* dfull = aempty + Sh::SA;                                 // [DB] a group's sums
    uint64_t* dempty = dfull + DB;
    uint64_t* done = dempty + DB;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kCopyWarp = kGemmSumWarps + kGemmConvWarps, kMmaWarp = kCopyWarp + 2;
    const int blocks = (p.n + 127) >> 7, tiles = (p.m + 127) >> 7;
    const int first = gemm_first(blocks * tiles, gridDim.x, blockIdx.x), end = gemm_first(blocks * tiles, gridDim.x, blockIdx.x + 1);
    const int steps = end - first;

    if (tid < Sh::NBars) {
        const int i = tid, w = 2 * Sh::SW, x = w + 2 * Sh::SX, a = x + 2 * Sh::SA, d = a + 2 * DB;
        mbar_init(wfull + i, i < Sh::SW ? 1 : i < w ? kGemmConvWarps / 2 : i < w + Sh::SX ? 1 : i < x ? 1 + kGemmSumWarps : i < x + Sh::SA ? kTeam : i < a ? 1 : i < a + DB ? 1 : i < d ? kGemmSumWarps : 1);
        fence_mbar_init();
        if (tid == 0) *fail = 0;
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Sh::TmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();                                   // (only the images' warp waits: weights are ready)
    auto wait = [&](uint64_t* bar, int parity) {               // false: it ran out (1 s)
        bool ok = mbar_try_wait(bar, (uint32_t)parity);
        if (!ok) ok = mbar_wait_bounded(bar, (uint32_t)parity);
        if (!ok) *fail = 1;
        return __all_sync(0xffffffffu, ok) != 0;
    };
    auto arrive_warp = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };

    if (warp == kCopyWarp || warp == kCopyWarp + 1) {
        const bool codes = warp == kCopyWarp;
        uint64_t *full = codes ? wfull : xfull, *empty = codes ? wempty : xempty;
        const int slots = codes ? Sh::SW : Sh::SX;
        if (!codes) pdl_wait();
        int kb = first % blocks, tile = first / blocks, i = 0, slot = 0, turn = 1;      // turn: parity of the slots' last emptying
        for (; i < steps; ++i) {
            if (i >= slots && !wait(&empty[slot], turn)) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(&full[slot], codes ? Sh::Packed : Sh::Image + Sh::Units);
                if (codes) tma_load_2d(sm + Sh::W + slot * Sh::Packed, &p.W, 64 * kb, 128 * tile, &full[slot]);
                else {
                    bulk_g2s(sm + Sh::X + slot * Sh::Image, p.images + (size_t)kb * Sh::Image, Sh::Image, &full[slot]);
                    bulk_g2s(sm + Sh::U + slot * Sh::Units, p.units + (size_t)kb * NT, Sh::Units, &full[slot]);
                }
            }
            if (++kb == blocks) { kb = 0; ++tile; }
            if (++slot == slots) { slot = 0; turn ^= 1; }
        }
        // no copy may be under way when the memory is given up
        __syncwarp();
        for (int j = max(i - slots, 0); j < i; ++j)
            if (!mbar_wait_bounded(&full[j % slots], (j / slots) & 1)) *fail = 1;
    } else if (warp == kMmaWarp) {
        const bool me = elect_lane();
        constexpr uint32_t id = umma_idesc_f16(NT, false, false);
        const uint64_t adesc = umma_desc_sw128(smem_u32(sm) + Sh::A), xdesc = umma_desc_sw128(smem_u32(sm) + Sh::X);
        for (int i = 0; i < steps; ++i) {
            const int sa = i % Sh::SA, sx = i % Sh::SX;
            if (!wait(&afull[sa], (i / Sh::SA) & 1) || !wait(&xfull[sx], (i / Sh::SX) & 1)) break;
            const uint64_t ad = adesc + (uint64_t)(sa * (Sh::Tile >> 4)), xd = xdesc + (uint64_t)(sx * (Sh::Image >> 4));
            bool ok = true;
#pragma unroll
            for (int g = 0; g < GS; ++g) {
                const int u = i * GS + g, b = u % DB;
                if (u >= DB) ok = ok && wait(&dempty[b], (u / DB - 1) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int e = 1; e >= 0; --e)
#pragma unroll
                    for (int j = 0; j < GROUP / 16; ++j) {
                        const int k = g * (GROUP / 16) + j;
                        const uint64_t a = ad + ((k >> 2) * 128 * 128 + 32 * (k & 3)) / 16;
                        const uint64_t x = xd + ((k >> 2) * (NT * 256) + e * (NT * 128) + 32 * (k & 3)) / 16;
                        if (e == 1 && j == 0) umma_f16<false>(me, tmem + b * NT, a, x, id);
                        else umma_f16<true>(me, tmem + b * NT, a, x, id);
                    }
                if (me) umma_commit(&dfull[b]);
            }
            if (!ok) break;
            if (me) {
                umma_commit(&aempty[sa]);
                umma_commit(&xempty[sx]);
            }
        }
        if (me) umma_commit(done);                             // also after a wait that ran out
        __syncwarp();
        if (!mbar_wait_bounded(done, 0)) *fail = 1;
    } else if (warp >= kGemmSumWarps) {
        // codes to f16, by two teams of four warps in turn, a step and a place of the operand each: a
        // thread four times 16 bytes (32 codes) of a row. A code c lies as c ^ 8 above 1024 in f16: 1032 + c
        const int ct = (tid - kGemmSumWarps * 32) % kTeam, chunk = ct & 3, r0 = ct >> 2, team = (warp - kGemmSumWarps) / (kTeam / 32);
        unsigned char* part = sm + Sh::A + team * Sh::Tile + (chunk >> 1) * (128 * 128);
        const bool turn = chunk & 2;                           // (halves two units apart: no bank conflicts)
        int sw = team, wturn = 0;
        for (int i = team; i < steps; i += 2) {
            if (!wait(&wfull[sw], wturn)) break;
            uint4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = lds128(sm + Sh::W + sw * Sh::Packed + (r0 + 32 * x) * 64 + 16 * chunk);
            if (i >= 2 && !wait(&aempty[team], ((i >> 1) - 1) & 1)) break;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = r0 + 32 * x;
                const uint32_t w[4] = {turn ? v[x].z : v[x].x, turn ? v[x].w : v[x].y, turn ? v[x].x : v[x].z, turn ? v[x].y : v[x].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int unit = 4 * (chunk & 1) + (turn ? j ^ 2 : j);
                    uint32_t r[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t z = (w[j] >> (4 * e) & 0x000f000fu) ^ 0x64086408u;
                        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&z), __half2half2(__ushort_as_half(0x6408)));
                        r[e] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    *reinterpret_cast<uint4*>(part + row * 128 + ((unit ^ (row & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
                }
            }
            fence_async_smem();
            mbar_arrive(&afull[team]);
            arrive_warp(&wempty[sw]);
            sw += 2;
            if (sw >= Sh::SW) { sw -= Sh::SW; wturn ^= 1; }
        }
    } else {
        // sums
        constexpr int C = NT / 2;                              // vectors of a thread
        const int quarter = warp & 3, c0 = (warp >> 2) * C, r = 32 * quarter + lane;
        const uint32_t trow = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)c0;
        const int groups = (p.n + GROUP - 1) / GROUP;
        int kb = first % blocks, tile = first / blocks;        // of the next step
        // of this thread's row in it, as they lie in memory (whatever is done with a load waits for it)
        auto scales = [&](uint32_t (&s)[GS]) {
            const int row = tile * 128 + r;
#pragma unroll
            for (int g = 0; g < GS; ++g) {
                s[g] = 0u;
                const size_t at = (size_t)row * p.lds + kb * GS + g;
                if (row < p.m && kb * GS + g < groups)
                    s[g] = BF16 ? static_cast<const uint16_t*>(p.scale)[at] : static_cast<const uint32_t*>(p.scale)[at];
            }
        };
        uint32_t next[2][GS];                                  // two steps ahead
        auto advance = [&]() {
            if (++kb == blocks) { kb = 0; ++tile; }
        };
        scales(next[0]);
        advance();
        scales(next[1]);
        f32x2 acc[C / 2];
#pragma unroll
        for (int x = 0; x < C / 2; ++x) acc[x] = 0ull;
        bool begun = first % blocks == 0;                      // this part has the row tile's first columns
        int at = first % blocks, rows = first / blocks;        // of this step
        int part = 0;
        for (int i = 0; i < steps; ++i) {
            const int sx = i % Sh::SX, row = rows * 128 + r;
            float s[GS];
#pragma unroll
            for (int g = 0; g < GS; ++g) {
                s[g] = BF16 ? __uint_as_float(next[0][g] << 16) : __uint_as_float(next[0][g]);
                next[0][g] = next[1][g];
            }
            advance();
            scales(next[1]);
            if (++at == blocks) { at = 0; ++rows; }
            if (!wait(&xfull[sx], (i / Sh::SX) & 1)) break;
            const float* un = reinterpret_cast<const float*>(sm + Sh::U + sx * Sh::Units) + c0;
            bool ok = true;
#pragma unroll
            for (int g = 0; g < GS; ++g) {
                const int u = i * GS + g, b = u % DB;
                ok = ok && wait(&dfull[b], (u / DB) & 1);
                if (!ok) break;
                tc_fence_after();
                uint32_t d[C];
                tmem_read(trow + b * NT, d);
#pragma unroll
                for (int x = 0; x < C / 2; x += 2) {
                    const float4 uu = *reinterpret_cast<const float4*>(un + 2 * x);
                    acc[x] = fma2(mul2(pack2(__uint_as_float(d[2 * x]), __uint_as_float(d[2 * x + 1])), pack2(uu.x, uu.y)), pack2(s[g], s[g]), acc[x]);
                    acc[x + 1] = fma2(mul2(pack2(__uint_as_float(d[2 * x + 2]), __uint_as_float(d[2 * x + 3])), pack2(uu.z, uu.w)), pack2(s[g], s[g]),
                                      acc[x + 1]);
                }
                tc_fence_before();
                arrive_warp(&dempty[b]);
            }
            if (!ok) break;
            arrive_warp(&xempty[sx]);
            if (at != 0 && i + 1 < steps) continue;
            // the end of the row tile, or of the share
            const bool whole = begun && at == 0;
            float* dst = whole ? p.y + row : p.part + ((size_t)blockIdx.x * 2 + part) * NT * 128 + r;
            const long long ld = whole ? p.ldy : 128;
            const float bias = whole && p.bias && row < p.m ? p.bias[row] : 0.0f;
            begun = true;
            part = 1;
#pragma unroll
            for (int x = 0; x < C / 2; ++x) {
                const float2 y = unpack2(mul2(acc[x], pack2(kGroupRoom, kGroupRoom)));
                acc[x] = 0ull;
                const int v = c0 + 2 * x;
                if (whole && row >= p.m) continue;
                if (v < p.T) dst[v * ld] = whole && p.bias ? fadd(y.x, bias) : y.x;
                if (v + 1 < p.T) dst[(v + 1) * ld] = whole && p.bias ? fadd(y.y, bias) : y.y;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Sh::TmemCols) : "memory");
    }
    // a wait that ran out: the outputs say so
    if (*fail) {
        const float nan = __int_as_float(0x7fffffff);
        for (int i = tid; i < 2 * NT * 128; i += kGemmThreads) p.part[(size_t)blockIdx.x * 2 * NT * 128 + i] = nan;
        for (int row = first / blocks * 128 + tid; row < min((end + blocks - 1) / blocks * 128, p.m); row += kGemmThreads)
            for (int v = 0; v < p.T; ++v) p.y[(size_t)v * p.ldy + row] = nan;
    }
}

// Adds the parts of row tiles that several CTAs have, in order of columns: grid (tiles, T).
template <int NT>
__global__ void __launch_bounds__(128) group_add_kernel(const __grid_constant__ GemmParams p, int ctas) {
    pdl_launch_dependents();
    pdl_wait();
    const int blocks = (p.n + 127) >> 7, tiles = (p.m + 127) >> 7, tile = blockIdx.x, v = blockIdx.y, row = tile * 128 + threadIdx.x;
    const int steps = blocks * tiles, first = tile * blocks;
    const int a = gemm_cta(steps, ctas, first), b = gemm_cta(steps, ctas, first + blocks - 1);
    if (a == b || row >= p.m) return;
    // only the first of the tile's CTAs can have begun before the tile: its part is its second then
    float y = p.part[(((size_t)a * 2 + (gemm_first(steps, ctas, a) < first)) * NT + v) * 128 + threadIdx.x];
#pragma unroll 4
    for (int c = a + 1; c <= b; ++c) y += p.part[((size_t)c * 2 * NT + v) * 128 + threadIdx.x];
    p.y[(size_t)v * p.ldy + row] = p.bias ? fadd(y, p.bias[row]) : y;
}

}  // namespace b2
