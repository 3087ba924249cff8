// tree_attn.cuh — attention of drafted tokens over the paged 8-bit KV cache and over their own
// f32 keys and values (sm_100a).
//
// A sequence's drafted rows see all of its cached keys, so nothing is masked there: the
// columns (row, head) of a KV head meet every tile of 128 keys. Both products run on the 5th-
// generation tensor cores in f16 with the factors that are f32 held as two f16 each:
//   x f = hi + lo, f a power of two that brings the largest to [2^13, 2^14)
// which keeps 22 bits of every element down to 2^-26 of the largest, and 2^-38 of the largest of
// those below. The cached codes are exact in f16; drafted keys and values are two
// f16 too, as keys j and 64 + j of a tile of their own, so that all four products are made.
//   S^T [key][column] = K Q^T      P: weights p x v_scale. Hi and lo of Q and P are columns side by
//   O^T [element][column] = V^T P  side (keys are read once: the MMAs are bound by reading operands)
// Keys and elements lie on the TMEM lanes: a thread has one key of a few columns, whose scales
// are its own. Each tile's output sums go to f32 registers, so that the tensor cores' sums stay
// short.
// A column's weights are relative to the largest p x v_scale of the keys that it sees, over all
// tiles: what a row does not see, or a key of large values and no probability, takes no bits
// from the others. For that the exponentials are relative to h, the largest score + exponent of the
// value scale, and an item's weights have one factor: 22 bits down to 2^-18 of that largest one, and
// an absolute 2^-30 of it below. Exponents count from that of the item's first tile of values, 2^-80
// to 2^80 times that, so that the sums of p stay in f32's range; a tile with values beyond has a
// factor of its own, which brings them back to there. h is a whole
// number and moves only when something is more than 2^8 above it: then the largest is found
// across the lanes; a tile that moves nothing needs no more than the warps' word that it does not.
//
// Measured (a call, us; bytes at 6.56 TB/s or operations at the bf16 rate allow the second figure):
//   1 sequence of 5 rows over 639 keys, 32 / 32 heads of 128             13   0.8  latency of one item
//   32 of 16 rows over 1152 keys, 32 / 32 heads of 128                  122    51  a tile's turn of the only place
//     for keys: conversion 1500 clocks, scores 600, waits between warps 800; issue slots 51 %
//   16 of up to 60 rows over up to 4000 keys, 32 / 8 heads of 128       209    18  the same with 64 columns
//   2 of 64 rows over 40000 keys, 32 / 4 heads of 64                    343    25  the softmax: 59 % of issue slots,
//     9.1 K instructions of warps a tile of 128 keys x 64 columns, tensor pipe active 20 %
// Two groups of softmax warps with every other tile each and two places for queries: 137 instead of 130.
#pragma once
#include <type_traits>

#include "f16_pairs.cuh"
#include "paged_rows.cuh"
#include "umma.cuh"

namespace b2 {

constexpr int kTreeRows = 64;

struct TreeAttnParams {
    PagedKv c;
    PagedRows r;             // kv_len: cached keys
    const long long* seen;   // [n_rows]
    const float* q;          // [n_rows][ldq], rotated and pre-scaled
    const float* k;          // [n_rows][ldk], rotated
    const float* v;          // [n_rows][ldv]
    float* out;              // [n_rows][ldo]
    long long ldq, ldk, ldv, ldo;
    int H, G;                // G = H / KVH
    int kc, nsplit;          // a split: kc cached keys (a multiple of 128), of which the last also has the
                             // drafted ones; nsplit: splits of cap keys
    float* part;             // [n_rows][H][nsplit][dh + 4]: o, m (base 2), l
    int* err;
};

__device__ __forceinline__ int tree_splits(int kc, int keys) { return max((keys - 1) / kc + 1, 1); }

// First the softmax warps: warp w reads TMEM lanes 32 (w % 4) .. + 31 and part w / 4 of a tile's
//   columns.
// Then the keys' warps: codes in shared memory to f16 operands; then the values', and an item's
//   queries. Drafted rows likewise. (Codes that waited in registers of these warps took 80
//   registers' worth of spills, and the fence behind the writes waits for loads under way.)
// One warp issues the MMAs. The last finds the items (a sequence's columns of a KV head against
//   a split of its keys) and their tiles' blocks, scales and factors (made by every softmax thread: 16
//   sequences of 32 / 8 heads of 128 217 us, now 208), up to eight tiles ahead, and asks for
//   the codes: a bulk copy for each block of 16 keys.
// A CTA a SM goes through its items with the pipeline running on from one to the next. Every
// wait is bounded; a warp whose wait ran out leaves its loop and sets the error word.
constexpr int kTreeRing = 8;
constexpr int kTreeKeys = 128;

enum { TREE_FIRST = 1, TREE_LAST = 2, TREE_DRAFT = 4, TREE_END = 8 };

struct TreeTile {
    int cell[8];             // block b of the tile in the pool (codes start at 16 dh times that; -1: none)
    float ks[8], vf[8];      // their scales, the values' times the tile's factor (-1 and 0: none),
    float ve[8];             // and the exponents of the values', from ref on
    float unit;              // what is one in the tile's output sums
    int ref;                 // the exponent of the item's first values that are not zeros (-127: none yet)
    int flags, item;
    int limit;               // keys of the tile
    int a, len, kvh;         // the item's rows and KV head,
    int col0, cols;          // its columns (row * G + head),
    int split, nsplit;
    int pad[4];
};

// DP: d_head rounded up to 64, 128 or 256; NC: columns of an item
template <int DP, int NC>
struct TreeShape {
    // (A second tile of keys in the place of two tiles of codes, d_head 128 and 16 columns: 153 us instead of 130.)
    static constexpr int KK = DP == 64 ? 2 : 1;                    // tiles of keys held,
    static constexpr int KV = DP == 64 || (DP == 128 && NC == 16) ? 2 : 1;      // of values,
    static constexpr int PB = DP == 256 ? 1 : 2;                   // of weights,
    static constexpr int ST = DP == 64 ? 6 : DP == 256 ? 1 : NC == 16 ? 4 : 2;  // and of codes as they come (keys, values, keys, ..)
    static constexpr int NB = ST < 2 ? 2 : ST;                     // barriers of those: a team's own
    static constexpr int Halves = DP / 64;                         // 128-byte parts of a row
    static constexpr int MH = DP == 256 ? 2 : 1;                   // 128 elements each of the output
    // Softmax warps: 8 for 16 columns (16, with 4 columns a thread: 32 sequences of 32 / 32 heads of 128 129 us,
    // now 123: what a warp does for a tile whatever its columns are costs issue slots), else 16 (8, with 32
    // columns a thread: two sequences of 40 K keys, 32 / 4 heads of 64: 400 us instead of 361)
    static constexpr int Soft = NC == 16 ? 8 : 16, Parts = Soft / 4;
    static constexpr int QC = NC / Parts;                          // columns of a thread
    // With 64 columns hi and lo go into the same sums, lo first: the MMAs take 96 clocks instead of 64 for
    // each 16 elements or keys, and the warps that read the sums have half as many to read (482 us, then 428). With
    // twice the elements the MMAs are more of a tile's time (32 / 8 heads of 128: 235 us, hi and lo in the same sums 256).
    static constexpr bool Same = DP == 64 && NC == 64;
    static constexpr int Sums = Same ? NC : 2 * NC;                // TMEM columns of a product
    // d_head up to 64: lanes 64 .. 127 of the output are the others again, so each has half of the columns
    static constexpr int OC = Same ? QC / 2 : QC;                  // columns of a thread's output
    // Warps that make operands of keys, of values: four each beside 8 softmax warps (eight: 130 us). Else two, but
    // four for values with only one place, which they refill between one tile's product and the next (16 sequences
    // of 32 / 8 heads of 128: 237 us with two, 211 with four; 32 / 4 heads of 64, two places: 361 and 369).
    static constexpr int KeyWarps = NC == 16 ? 4 : 2, ValueWarps = NC == 16 || KV == 1 ? 4 : 2;
    static constexpr int Threads = (Soft + KeyWarps + ValueWarps + 2) * 32;
    static constexpr int Tile = Halves * kTreeKeys * 128;          // [part][key][64 f16], swizzled
    static constexpr int QPart = Halves * 2 * NC * 128;            // [part][column: hi, lo][64 f16], swizzled
    static constexpr int PPart = kTreeKeys * 128;                  // [key][64 columns: hi, lo], swizzled
    static constexpr int PParts = 2 * NC > 64 ? 2 : 1;
    static constexpr int K = 0;
    static constexpr int V = K + KK * Tile;
    static constexpr int Q = V + KV * Tile;
    static constexpr int P = Q + QPart;
    static constexpr int Codes = P + PB * PParts * PPart;          // [block][16 keys][dh]
    static constexpr int Ring = Codes + ST * kTreeKeys * DP;
    static constexpr int Unit = Ring + kTreeRing * (int)sizeof(TreeTile);       // [ring][NC] f32: of a column's scores
    static constexpr int Seen = Unit + kTreeRing * NC * 4;         // [ring][NC] words
    static constexpr int Dks = Seen + kTreeRing * NC * 8;          // [ring][64] scales of drafted keys
    static constexpr int Dvs = Dks + kTreeRing * 64 * 4;           // and values
    static constexpr int Moves = Dvs + kTreeRing * 64 * 4;         // [2][4 parts] 1 + the last tile that moves h
    static constexpr int Xm = Moves + 8 * 4;                       // [2][4 parts][4][QC] largest scores
    static constexpr int Xl = Xm + 2 * 16 * QC * 4;                // [4][4][QC] sums
    static constexpr int Bs = Xl + 16 * QC * 4;                    // [16 warps][QC] -h
    static constexpr int Bd = Bs + 16 * QC * 4;                    // [16][QC] how far it moves; at the end 1 / sum
    static constexpr int Bk = Bd + 16 * QC * 4;                    // [2][16][QC] the factor of what was before: its root
    static constexpr int Bars = Bk + 2 * 16 * QC * 4;
    static constexpr int NBars = 2 * kTreeRing + 2 * NB + 2 * KK + 2 * KV + 2 + 4 + 2 + 4 + 4 + 1 + 1;
    static constexpr int Bytes = Bars + NBars * 8 + 16;
    static constexpr int Alloc = Bytes + 1024;                     // operands start on 1024 bytes
    static constexpr int TmemS = 0, TmemO = 2 * Sums;              // two buffers each
    static constexpr int TmemUsed = 2 * Sums + 2 * MH * Sums, TmemCols = TmemUsed <= 128 ? 128 : TmemUsed <= 256 ? 256 : 512;
    static_assert(TmemUsed <= 512 && Alloc <= 227 * 1024, "");
};

// eight codes of two words as f16: 1024 + (code + 128) by bytes, less 1152
__device__ __forceinline__ uint4 codes_f16(uint32_t a, uint32_t b) {
    const uint32_t x = a ^ 0x80808080u, y = b ^ 0x80808080u;
    uint32_t r[4] = {__byte_perm(x, 0x64646464u, 0x4140), __byte_perm(x, 0x64646464u, 0x4342),
                     __byte_perm(y, 0x64646464u, 0x4140), __byte_perm(y, 0x64646464u, 0x4342)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r[i]), __half2half2(__ushort_as_half(0x6480)));
        r[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

constexpr int kWeightBits = 5;                     // (weights: p x v_scale may reach 2^(kMoveBits + 1.5))
constexpr float kMoveBits = 8.0f;
constexpr int kValueBits = 80;                     // how far h follows the exponents of value scales
constexpr float kDraftedUnit = 64.0f;              // a drafted row's f16 reach 2^14, codes 2^7: brings its scale to theirs but for a bit

// the exponent of a scale (>= 0; -127 for 0), and from `ref` on as far as h follows
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23 & 0xff) - 127; }
__device__ __forceinline__ int value_exponent(float scale, int ref) { return min(max(exponent_of(scale) - ref, -kValueBits), kValueBits); }

__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

// A row of DP f32 elements, 16 lanes, lane l16 the elements 4 l16 + 64 i ..
template <int DP>
__device__ __forceinline__ void load_row(float4 (&x)[DP / 64], const float* src, bool live, int dh, int l16) {
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
        x[i] = live && 4 * l16 + 64 * i < dh ? *reinterpret_cast<const float4*>(src + 4 * l16 + 64 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// The row as hi and lo at hi_at(i, unit) and lo_at: the 16-byte unit of part i. Returns the scale of
// its values: NaN for a row that is not finite (its elements are zeros then, so that they harm
// no one else).
template <int DP, typename At>
__device__ __forceinline__ float put_row_f16(float4 (&x)[DP / 64], int l16, At hi_at, At lo_at) {
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        bad |= x[i].x != x[i].x || x[i].y != x[i].y || x[i].z != x[i].z || x[i].w != x[i].w;
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float f, unit;
    f16_factor(top, kRowBits, f, unit);
    const bool fine = top < INFINITY;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        uint2 hi, lo;
        if (!fine) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        split_f16(x[i].x * f, x[i].y * f, hi.x, lo.x);
        split_f16(x[i].z * f, x[i].w * f, hi.y, lo.y);
        *reinterpret_cast<uint2*>(hi_at(i, l16 >> 1) + 8 * (l16 & 1)) = hi;
        *reinterpret_cast<uint2*>(lo_at(i, l16 >> 1) + 8 * (l16 & 1)) = lo;
    }
    return fine ? unit : __int_as_float(0x7fffffff);
}

template <int DP, int NC>
__global__ void __launch_bounds__((TreeShape<DP, NC>::Threads), 1) tree_attn_kernel(const __grid_constant__ TreeAttnParams p) {
    using Sh = TreeShape<DP, NC>;
    constexpr int KK = Sh::KK, KV = Sh::KV, PB = Sh::PB, ST = Sh::ST, NB = Sh::NB, QC = Sh::QC, OC = Sh::OC, MH = Sh::MH, Sums = Sh::Sums;
    constexpr bool Same = Sh::Same;
    extern __shared__ unsigned char ta_raw[];
    unsigned char* sm = ta_raw + ((1024u - (smem_u32(ta_raw) & 1023u)) & 1023u);
    TreeTile* ring = reinterpret_cast<TreeTile*>(sm + Sh::Ring);
    uint64_t* tready = reinterpret_cast<uint64_t*>(sm + Sh::Bars);     // [ring] a tile is described
    uint64_t* tfree = tready + kTreeRing;                              // [ring] and not needed any more
    uint64_t* cfull = tfree + kTreeRing;                               // [NB] codes have come
    uint64_t* cempty = cfull + NB;                                     // [NB] and are turned
    uint64_t* kfull = cempty + NB;                                     // [KK] keys written
    uint64_t* kempty = kfull + KK;                                     // [KK] their scores are made
    uint64_t* vfull = kempty + KK;                                     // [KV]
    uint64_t* vempty = vfull + KV;                                     // [KV]
    uint64_t* qfull = vempty + KV;                                     // an item's queries written
    uint64_t* qfree = qfull + 1;                                       // its last scores made
    uint64_t* sfull = qfree + 1;                                       // [2] scores in TMEM
    uint64_t* sfree = sfull + 2;                                       // [2] read
    uint64_t* pfull = sfree + 2;                                       // [2] weights written
    uint64_t* ofull = pfull + 2;                                       // [2] output sums in TMEM (weights read)
    uint64_t* ofree = ofull + 2;                                       // [2] read
    uint64_t* part_bar = ofree + 2;                                    // [4] the warps of a column part meet
    uint64_t* all_bar = part_bar + 4;                                  // all softmax warps meet
    uint64_t* done = all_bar + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int dh = p.c.dh;
    constexpr int kMmaWarp = Sh::Soft + Sh::KeyWarps + Sh::ValueWarps, kPlanWarp = kMmaWarp + 1;

    after_previous();
    if (tid == 0) {
        for (int i = 0; i < kTreeRing; ++i) { mbar_init(&tready[i], 1); mbar_init(&tfree[i], Sh::Soft + Sh::KeyWarps + Sh::ValueWarps + 1); }
        for (int i = 0; i < NB; ++i) { mbar_init(&cfull[i], 1); mbar_init(&cempty[i], i & 1 ? Sh::ValueWarps : Sh::KeyWarps); }
        for (int i = 0; i < KK; ++i) { mbar_init(&kfull[i], Sh::KeyWarps); mbar_init(&kempty[i], 1); }
        for (int i = 0; i < KV; ++i) { mbar_init(&vfull[i], Sh::ValueWarps); mbar_init(&vempty[i], 1); }
        mbar_init(qfull, Sh::ValueWarps); mbar_init(qfree, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sfull[i], 2); mbar_init(&sfree[i], Sh::Soft);
            mbar_init(&ofull[i], 1); mbar_init(&ofree[i], Sh::Soft);
            mbar_init(&pfull[i], Sh::Soft);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&part_bar[i], 4);
        mbar_init(all_bar, Sh::Soft); mbar_init(done, 1);
        fence_mbar_init();
        *fail = 0;
    }
    if (tid < 8) reinterpret_cast<int*>(sm + Sh::Moves)[tid] = 0;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Sh::TmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // bounded (1 s); `pause` ns between polls, which take issue slots from the warps that work.
    // false: it ran out, and the caller leaves its loop
    auto wait = [&](uint64_t* bar, int parity, unsigned pause) {
        if (mbar_try_wait(bar, (uint32_t)parity)) return true;
        const uint64_t t0 = globaltimer_ns();
        for (unsigned k = 1; !mbar_try_wait(bar, (uint32_t)parity); ++k) {
            __nanosleep(pause);
            if ((k & 63u) == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
                *fail = 1;
                return false;
            }
        }
        return true;
    };
    auto wait_warp = [&](uint64_t* bar, int parity, unsigned pause) { return __all_sync(0xffffffffu, wait(bar, parity, pause)) != 0; };
    auto arrive_warp = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    auto ring_parity = [](int t) { return (t / kTreeRing) & 1; };

    if (warp == kPlanWarp) {
        // ---- items and tiles
        const int group = lane >> 3, b = lane & 7, psz = 1 << p.c.page_log2;
        int t = 0, base = 0, come = 0;                         // come: tiles of codes asked for
        unsigned item = blockIdx.x, before = 0;                // items of the sequences before `base`
        bool ok = true;
        for (int n = 0; ok; ++n, item += gridDim.x) {
            // the item's sequence: 32 at a time
            int s = -1, a = 0, len = 0, kv = 0;
            unsigned idx = 0;
            while (base < p.r.n_seq) {
                SeqRows q{0, 0, 0};
                unsigned cnt = 0;
                if (base + lane < p.r.n_seq) {
                    q = seq_rows(p.r, base + lane);
                    if (q.len > kTreeRows) set_err(p.err, B2_DEV_ERR_TOO_MANY);
                    else if (q.len > 0) {
                        if (q.kv > p.r.cap) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
                        cnt = (unsigned)(((q.len * p.G + NC - 1) / NC) * p.c.KVH * tree_splits(p.kc, min(q.kv, p.r.cap)));
                    }
                }
                unsigned incl = cnt;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                const unsigned total = __shfl_sync(0xffffffffu, incl, 31);
                if (item - before < total) {
                    const int src = __ffs(__ballot_sync(0xffffffffu, incl > item - before)) - 1;
                    idx = item - before - __shfl_sync(0xffffffffu, incl - cnt, src);
                    s = base + src;
                    a = __shfl_sync(0xffffffffu, q.a, src);
                    len = __shfl_sync(0xffffffffu, q.len, src);
                    kv = min(__shfl_sync(0xffffffffu, q.kv, src), p.r.cap);
                    break;
                }
                before += total;
                base += 32;
            }
            if (s < 0) {
                if (t >= kTreeRing) ok = wait_warp(&tfree[t & (kTreeRing - 1)], ring_parity(t) ^ 1, 100);
                if (ok) {
                    if (lane == 0) ring[t & (kTreeRing - 1)].flags = TREE_END;
                    arrive_warp(&tready[t & (kTreeRing - 1)]);
                }
                break;
            }
            // column tiles first: CTAs that run at once read the same keys
            const int ctiles = (len * p.G + NC - 1) / NC, nsplit = tree_splits(p.kc, kv);
            const int ct = (int)(idx % (unsigned)ctiles), rest = (int)(idx / (unsigned)ctiles), kvh = rest % p.c.KVH;
            const int split = min(rest / p.c.KVH, nsplit - 1);  // (row ranges that overlap could count past 32 bits)
            const int j0 = split * p.kc, jend = kv - j0 < p.kc ? kv : j0 + p.kc;
            const int ntiles = (max(jend - j0, 0) + kTreeKeys - 1) / kTreeKeys, all = ntiles + (split == nsplit - 1);
            int ref = -127;
            for (int i0 = 0; i0 < all && ok; i0 += 4) {
                const int i = i0 + group, in = i * kTreeKeys + 16 * b, cnt = min(all - i0, 4);
                int cell = -1;
                float ks = -1.0f, vs = 0.0f;
                if (i < ntiles && in < jend - j0) {
                    const int j = j0 + in, page = page_of(p.c, p.r, s, j);
                    if (page < 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
                    else {
                        cell = (page * p.c.KVH + kvh) * (psz >> 4) + ((j & (psz - 1)) >> 4);
                        ks = p.c.ks[cell];
                        vs = p.c.vs[cell];
                    }
                }
                float vtop = vs;
#pragma unroll
                for (int o = 4; o >= 1; o >>= 1) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, o));
                if (ref == -127) {
                    const unsigned any = __ballot_sync(0xffffffffu, vtop > 0.0f);
                    if (any) ref = exponent_of(__shfl_sync(0xffffffffu, vtop, __ffs(any) - 1));
                }
                float f, unit;
                f16_factor(vtop, kWeightBits + value_exponent(vtop, ref), f, unit);     // (the same for all tiles but those of extreme scales)
                for (int u = 0; u < cnt && ok; ++u)
                    if (t + u >= kTreeRing) ok = wait_warp(&tfree[(t + u) & (kTreeRing - 1)], ring_parity(t + u) ^ 1, 100);
                if (!ok) break;
                if (group < cnt) {
                    TreeTile& d = ring[(t + group) & (kTreeRing - 1)];
                    d.cell[b] = cell; d.ks[b] = ks; d.vf[b] = vs * f; d.ve[b] = (float)value_exponent(vs, ref);
                    if (b == 0) {
                        d.flags = (i == 0 ? TREE_FIRST : 0) | (i == all - 1 ? TREE_LAST : 0) | (i == ntiles ? TREE_DRAFT : 0);
                        d.item = n; d.limit = jend - j0 - i * kTreeKeys;
                        d.a = a; d.len = len; d.kvh = kvh; d.col0 = ct * NC; d.cols = min(len * p.G - ct * NC, NC);
                        d.split = split; d.nsplit = nsplit;
                        d.unit = unit; d.ref = ref;
                    }
                }
                __syncwarp();
                if (lane < cnt) mbar_arrive(&tready[(t + lane) & (kTreeRing - 1)]);
                t += cnt;
                // the tiles' codes: a bulk copy a block
                for (int u = 0; u < cnt && i0 + u < ntiles; ++u) {
                    const int c = __shfl_sync(0xffffffffu, cell, 8 * u + b);
                    const bool mine = group == 0 && c >= 0;
                    const unsigned bytes = __popc(__ballot_sync(0xffffffffu, mine)) * kKvBlock * dh;
#pragma unroll
                    for (int v = 0; v < 2; ++v, ++come) {
                        const int slot = come % ST;
                        if (come >= ST) ok = ok && wait_warp(&cempty[(come - ST) % NB], ((come - ST) / NB) & 1, 50);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&cfull[come % NB], bytes);
                        __syncwarp();
                        if (mine)
                            bulk_g2s(sm + Sh::Codes + slot * kTreeKeys * DP + b * kKvBlock * dh, (v ? p.c.v : p.c.k) + (size_t)c * kKvBlock * dh,
                                     kKvBlock * dh, &cfull[come % NB]);
                    }
                    if (!ok) break;
                }
            }
        }
        // no copy may be under way when the memory is given up
        for (int c = max(come - ST, 0); c < come; ++c)
            if (!mbar_wait_bounded(&cfull[c % NB], (c / NB) & 1)) *fail = 1;
    } else if (warp == kMmaWarp) {
        // ---- MMAs
        const bool me = elect_lane();
        const uint32_t base = smem_u32(sm);
        constexpr uint32_t ids = umma_idesc_f16(Sums, false, false), ido = umma_idesc_f16(Sums, true, true);
        const uint64_t kdesc = umma_desc_sw128(base + Sh::K), qdesc = umma_desc_sw128(base + Sh::Q);
        // (d_head 64: lanes 64 .. 127 of the output repeat the others)
        const uint64_t vdesc = umma_desc_sw128_mn(base + Sh::V, Sh::Halves > 1 ? kTreeKeys * 128 : 0);
        const uint64_t pdesc = umma_desc_sw128_mn(base + Sh::P, !Same && Sh::PParts > 1 ? Sh::PPart : 0);
        bool ok = true;
        int items = 0;
        auto scores = [&](int t, int flags) {
            const int slot = t % KK, use = t / KK;
            ok = ok && wait_warp(&kfull[slot], use & 1, 20);
            if (ok && (flags & TREE_FIRST)) ok = wait_warp(qfull, items & 1, 20);
            if (ok && t > 1) ok = wait_warp(&sfree[t & 1], ((t >> 1) - 1) & 1, 20);
            if (!ok) return;
            tc_fence_after();
            const uint64_t kd = kdesc + (uint64_t)(slot * (Sh::Tile >> 4));
            const uint32_t to = tmem + Sh::TmemS + (t & 1) * Sums;
#pragma unroll
            for (int lo = Same; lo >= 0; --lo)
#pragma unroll
                for (int i = 0; i < 4 * Sh::Halves; ++i) {
                    const uint64_t a = kd + ((i >> 2) * (kTreeKeys * 128) + 32 * (i & 3)) / 16;
                    const uint64_t b = qdesc + ((i >> 2) * (2 * NC * 128) + lo * NC * 128 + 32 * (i & 3)) / 16;
                    if (lo == Same && i == 0) umma_f16<false>(me, to, a, b, ids);
                    else umma_f16<true>(me, to, a, b, ids);
                }
            if (me) {
                umma_commit(&kempty[slot]);
                if (flags & TREE_LAST) umma_commit(qfree);
                umma_commit(&sfull[t & 1]);
            }
            if (flags & TREE_LAST) ++items;
            // drafted values' scales come with the values
            if (flags & TREE_DRAFT) ok = wait_warp(&vfull[t % KV], (t / KV) & 1, 20);
            if (me) mbar_arrive(&sfull[t & 1]);                // passes on what the others wrote: units, scales
        };
        auto output = [&](int t) {
            const int slot = t % KV, use = t / KV;
            ok = ok && wait_warp(&pfull[t & 1], (t >> 1) & 1, 20) && wait_warp(&vfull[slot], use & 1, 20);
            if (ok && t > 1) ok = wait_warp(&ofree[t & 1], ((t >> 1) - 1) & 1, 20);
            if (!ok) return;
            tc_fence_after();
            const uint64_t pd = pdesc + (uint64_t)(t % PB * (Sh::PParts * Sh::PPart >> 4));
#pragma unroll
            for (int mh = 0; mh < MH; ++mh) {
                const uint64_t vd = vdesc + (uint64_t)(slot * (Sh::Tile >> 4) + mh * (2 * kTreeKeys * 128 >> 4));
                const uint32_t to = tmem + Sh::TmemO + ((t & 1) * MH + mh) * Sums;
#pragma unroll
                for (int lo = Same; lo >= 0; --lo)
#pragma unroll
                    for (int k = 0; k < kTreeKeys / 16; ++k) {
                        const uint64_t b = pd + (lo * Sh::PPart + k * 2048) / 16;
                        if (lo == Same && k == 0) umma_f16<false>(me, to, vd, b, ido);
                        else umma_f16<true>(me, to, vd + k * (2048 / 16), b, ido);
                    }
            }
            if (me) {
                umma_commit(&vempty[slot]);
                umma_commit(&ofull[t & 1]);
            }
        };
        // the flags of tile t; its description is not needed after that
        auto flags_of = [&](int t) {
            ok = ok && wait_warp(&tready[t & (kTreeRing - 1)], ring_parity(t), 20);
            const int f = ok ? ring[t & (kTreeRing - 1)].flags : TREE_END;
            if (ok) arrive_warp(&tfree[t & (kTreeRing - 1)]);
            return f;
        };
        int flags = flags_of(0);
        if (!(flags & TREE_END)) scores(0, flags);
        for (int t = 0; ok && !(flags & TREE_END); ++t) {
            flags = flags_of(t + 1);
            // the next tile's scores go first, except those of another item, whose queries
            // wait for this one's, and drafted ones where their values wait for the only place
            const bool ahead = !(flags & (TREE_END | TREE_FIRST)) && !(KV == 1 && (flags & TREE_DRAFT));
            if (ahead) scores(t + 1, flags);
            output(t);
            if (!ahead && !(flags & TREE_END)) scores(t + 1, flags);
        }
        if (me) umma_commit(done);                             // also after a wait that ran out: no MMA may be
        __syncwarp();
        if (!mbar_wait_bounded(done, 0)) *fail = 1;            // under way when its memory is given up
    } else if (warp >= Sh::Soft) {
        // ---- operands: a team for the keys, one for the values
        constexpr int Chunks = DP / 16;                        // 16 codes each of a row
        constexpr int Wide = kTreeKeys * Chunks / (32 * Sh::ValueWarps) < 8 ? kTreeKeys * Chunks / (32 * Sh::ValueWarps) : 8;
        const bool keys = warp < Sh::Soft + Sh::KeyWarps;
        const int team = 32 * (keys ? Sh::KeyWarps : Sh::ValueWarps), step = team / Chunks, lines = team / 16;
        const int ct = tid - (Sh::Soft + (keys ? 0 : Sh::KeyWarps)) * 32, chunk = ct % Chunks, key0 = ct / Chunks;
        const float* rows = keys ? p.k : p.v;
        const long long ldr = keys ? p.ldk : p.ldv;
        unsigned char* tiles = sm + (keys ? Sh::K : Sh::V);
        uint64_t *full = keys ? kfull : vfull, *empty = keys ? kempty : vempty;
        float* scales = reinterpret_cast<float*>(sm + (keys ? Sh::Dks : Sh::Dvs));
        // a tile's codes (blocks that are not there: some others, which count nothing) as f16
        auto put = [&](const unsigned char* codes, unsigned char* tile) {
            unsigned char* part = tile + (chunk >> 2) * kTreeKeys * 128;
            const int u0 = 2 * (chunk & 3), turn = (chunk >> 2) & 1;      // (parts in turn: no bank conflicts)
            const bool in = 16 * chunk < dh;
#pragma unroll 1
            for (int at = key0; at < kTreeKeys; at += Wide * step) {
                uint4 r[Wide];
#pragma unroll
                for (int x = 0; x < Wide; ++x) r[x] = in ? lds128(codes + (at + x * step) * dh + 16 * chunk) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int x = 0; x < Wide; ++x) {
                    const int key = at + x * step;
                    const uint4 a = codes_f16(turn ? r[x].z : r[x].x, turn ? r[x].w : r[x].y), b = codes_f16(turn ? r[x].x : r[x].z, turn ? r[x].y : r[x].w);
                    unsigned char* row = part + key * 128;
                    *reinterpret_cast<uint4*>(row + (((u0 + turn) ^ (key & 7)) << 4)) = a;
                    *reinterpret_cast<uint4*>(row + (((u0 + 1 - turn) ^ (key & 7)) << 4)) = b;
                }
            }
        };
        constexpr int Batch = 8 / (DP / 64);                   // rows of a lane group in flight
        // drafted rows: key j and 64 + j of the tile, all loads of a batch first. (What lies past the
        // last one is some other tile's: its scores are masked, its values are finite.)
        auto put_drafted = [&](unsigned char* tile, const TreeTile& d, float* scale) {
            for (int r0 = 0; r0 < d.len; r0 += lines * Batch) {
                float4 x[Batch][DP / 64];
#pragma unroll
                for (int b = 0; b < Batch; ++b) {
                    const int j = r0 + lines * b + (ct >> 4);
                    load_row<DP>(x[b], rows + (size_t)(d.a + min(j, d.len - 1)) * ldr + (size_t)d.kvh * dh, j < d.len, dh, ct & 15);
                }
#pragma unroll
                for (int b = 0; b < Batch; ++b) {
                    const int j = r0 + lines * b + (ct >> 4);
                    if (r0 + lines * b >= d.len) break;        // (whole warps)
                    auto at = [&](int row) {
                        return [=](int i, int u) { return tile + i * kTreeKeys * 128 + row * 128 + ((u ^ (row & 7)) << 4); };
                    };
                    const float unit = put_row_f16<DP>(x[b], ct & 15, at(j), at(64 + j));
                    if ((ct & 15) == 0) scale[j] = unit;
                }
            }
        };
        auto put_queries = [&](const TreeTile& d) {
            const int it = d.item & (kTreeRing - 1);
            float* unit = reinterpret_cast<float*>(sm + Sh::Unit) + it * NC;
            long long* seen = reinterpret_cast<long long*>(sm + Sh::Seen) + it * NC;
            for (int c0 = 0; c0 < d.cols; c0 += lines * Batch) {
                float4 x[Batch][DP / 64];
#pragma unroll
                for (int b = 0; b < Batch; ++b) {
                    const int c = c0 + lines * b + (ct >> 4), cc = d.col0 + min(c, d.cols - 1);
                    load_row<DP>(x[b], p.q + (size_t)(d.a + cc / p.G) * p.ldq + (size_t)(d.kvh * p.G + cc % p.G) * dh, c < d.cols, dh, ct & 15);
                }
#pragma unroll
                for (int b = 0; b < Batch; ++b) {
                    const int c = c0 + lines * b + (ct >> 4);
                    if (c0 + lines * b >= d.cols) break;       // (whole warps)
                    auto at = [&](int col) {
                        return [=](int i, int u) { return sm + Sh::Q + i * 2 * NC * 128 + col * 128 + ((u ^ (col & 7)) << 4); };
                    };
                    const float un = put_row_f16<DP>(x[b], ct & 15, at(c), at(NC + c));
                    if ((ct & 15) == 0) {
                        unit[c] = un * 1.4426950408889634f;    // log2 e
                        seen[c] = c < d.cols ? p.seen[d.a + (d.col0 + c) / p.G] : 0;
                    }
                }
            }
        };
        if (!keys) {                                           // what nothing has written yet are zeros
            for (int i = ct; i < KV * Sh::Tile / 16; i += team) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0u, 0u, 0u, 0u);
            for (int i = ct; i < Sh::QPart / 16; i += team) reinterpret_cast<uint4*>(sm + Sh::Q)[i] = make_uint4(0u, 0u, 0u, 0u);
            for (int i = ct; i < kTreeRing * NC; i += team) {
                reinterpret_cast<float*>(sm + Sh::Unit)[i] = 0.0f;
                reinterpret_cast<long long*>(sm + Sh::Seen)[i] = 0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * Sh::ValueWarps) : "memory");      // (nobody has waited for anything yet)
        }
        bool ok = true;
        for (int t = 0, come = keys ? 0 : 1; ok; ++t) {
            ok = wait_warp(&tready[t & (kTreeRing - 1)], ring_parity(t), 50);
            if (!ok) break;
            const TreeTile& d = ring[t & (kTreeRing - 1)];
            if (d.flags & TREE_END) break;
            const int slots = keys ? KK : KV, slot = t % slots;
            if (!keys && (d.flags & TREE_FIRST)) {
                if (d.item > 0) ok = wait_warp(qfree, (d.item - 1) & 1, 50);
                if (!ok) break;
                put_queries(d);
                fence_async_smem();
                arrive_warp(qfull);
            }
            unsigned char* tile = tiles + slot * Sh::Tile;
            if (d.flags & TREE_DRAFT) {
                if (t >= slots) ok = wait_warp(&empty[slot], (t / slots - 1) & 1, 50);
                if (!ok) break;
                put_drafted(tile, d, scales + (t & (kTreeRing - 1)) * 64);
            } else {
                const int cs = come % ST;
                ok = wait_warp(&cfull[come % NB], (come / NB) & 1, 50);
                if (ok && t >= slots) ok = wait_warp(&empty[slot], (t / slots - 1) & 1, 50);
                if (!ok) break;
                put(sm + Sh::Codes + cs * kTreeKeys * DP, tile);
                arrive_warp(&cempty[come % NB]);
                come += 2;
            }
            fence_async_smem();
            arrive_warp(&full[slot]);
            arrive_warp(&tfree[t & (kTreeRing - 1)]);
        }
    } else {
        // ---- softmax and output
        const int quarter = warp & 3, part = warp >> 2, key = 32 * quarter + lane;
        const uint32_t trow = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(part * QC);
        float* bs = reinterpret_cast<float*>(sm + Sh::Bs) + warp * QC;
        float* bk = reinterpret_cast<float*>(sm + Sh::Bk) + warp * QC;
        float* bd = reinterpret_cast<float*>(sm + Sh::Bd) + warp * QC;
        float* xm = reinterpret_cast<float*>(sm + Sh::Xm) + part * 4 * QC;
        float* xl = reinterpret_cast<float*>(sm + Sh::Xl) + part * 4 * QC;
        int met = 0, met_all = 0;                              // how often the part's warps, all of them have met
        bool ok = true;
        auto meet = [&]() {
            arrive_warp(&part_bar[part]);
            ok = wait_warp(&part_bar[part], met++ & 1, 20);
            return ok;
        };
        // the sums of n columns
        auto read_sums = [&](uint32_t at, f32x2* y, auto n) {
            constexpr int N = decltype(n)::value, M = Same ? N / 2 : N < 8 ? N : 8;
#pragma unroll
            for (int i = 0; i < (Same ? 1 : N / M); ++i) {
                uint32_t c[M], z[M];
                tmem_read2(at + i * M, at + (Same ? M : NC + i * M), c, z);
#pragma unroll
                for (int x = 0; x < M / 2; ++x) {
                    const f32x2 a = pack2(__uint_as_float(c[2 * x]), __uint_as_float(c[2 * x + 1]));
                    const f32x2 b = pack2(__uint_as_float(z[2 * x]), __uint_as_float(z[2 * x + 1]));
                    if constexpr (Same) { y[x] = a; y[M / 2 + x] = b; }
                    else y[i * M / 2 + x] = add2(a, b);
                }
            }
        };
        const int oc0 = OC < QC ? (quarter >> 1) * OC : 0, oelem = OC < QC ? key & 63 : key;      // of the thread's output
        int* moves = reinterpret_cast<int*>(sm + Sh::Moves) + part;
        float h = 0.0f;                                        // of column `lane`,
        bool unset = true;                                     // which has seen no key yet
        f32x2 l[QC / 2], o[MH][OC / 2];
        // Output sums are folded two tiles later, when their products are surely made; with one buffer of
        // weights one tile later, before they are written.
        // output sums of tile t; u: what a unit of them is, moved: whether that tile moved h
        auto fold = [&](int t, float u, bool moved) {
            ok = ok && wait_warp(&ofull[t & 1], (t >> 1) & 1, 20);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int mh = 0; mh < MH; ++mh) {
                if (moved) {
#pragma unroll
                    for (int x = 0; x < OC / 2; ++x) {
                        const float2 bb = *reinterpret_cast<const float2*>(bk + (t & 1) * 16 * QC + oc0 + 2 * x);
                        o[mh][x] = mul2(mul2(o[mh][x], pack2(bb.x, bb.y)), pack2(bb.x, bb.y));
                    }
                }
                f32x2 y[OC / 2];
                read_sums(trow + Sh::TmemO + ((t & 1) * MH + mh) * Sums + oc0, y, std::integral_constant<int, OC>{});
#pragma unroll
                for (int x = 0; x < OC / 2; ++x) o[mh][x] = fma2(y[x], pack2(u, u), o[mh][x]);
            }
            tc_fence_before();
            arrive_warp(&ofree[t & 1]);
        };
        // where a column's output goes: its row of `out`, or its partial result
        auto column_out = [&](const TreeTile& d, int col) {
            const int cc = d.col0 + col, tok = cc / p.G, row = d.a + tok, head = d.kvh * p.G + cc - tok * p.G;
            return d.nsplit > 1 ? p.part + (((size_t)row * p.H + head) * p.nsplit + d.split) * (dh + 4)
                                : p.out + (size_t)row * p.ldo + (size_t)head * dh;
        };
        float u1 = 0.0f, u2 = 0.0f;                            // of the two tiles whose output is pending
        bool moved1 = false, moved2 = false;
        int begun = 0;                                         // tiles of the item before this one
        for (int t = 0; ok; ++t, ++begun) {
            if (!wait_warp(&tready[t & (kTreeRing - 1)], ring_parity(t), 20)) break;
            const TreeTile& d = ring[t & (kTreeRing - 1)];
            const int flags = d.flags;
            if (flags & TREE_END) break;
            const bool draft = flags & TREE_DRAFT, first = flags & TREE_FIRST;
            if (first) {
                begun = 0;
                h = 0.0f;
                unset = lane < QC && part * QC + lane < d.cols;
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) l[x] = 0ull;
#pragma unroll
                for (int mh = 0; mh < MH; ++mh)
#pragma unroll
                    for (int x = 0; x < OC / 2; ++x) o[mh][x] = 0ull;
                if (lane < QC) bs[lane] = 0.0f;
                __syncwarp();
            }
            const int it = d.item & (kTreeRing - 1);
            const float* unit = reinterpret_cast<const float*>(sm + Sh::Unit) + it * NC + part * QC;
            if (!wait_warp(&sfull[t & 1], (t >> 1) & 1, 20)) break;
            tc_fence_after();
            f32x2 s[QC / 2];
            read_sums(trow + Sh::TmemS + (t & 1) * Sums, s, std::integral_constant<int, QC>{});
            tc_fence_before();
            arrive_warp(&sfree[t & 1]);
            // this key's scale, its value scale's exponent and that with the factor of the tile's weights
            float ks, vf, ve, un;
            bool gone;
            if (!draft) {
                ks = d.ks[key >> 4];
                vf = d.vf[key >> 4];
                ve = d.ve[key >> 4];
                un = d.unit;
                gone = ks < 0.0f || key >= d.limit;
            } else {
                if (begun >= PB) PB == 2 ? fold(t - 2, u2, moved2) : fold(t - 1, u1, moved1);
                if (!ok) break;
                const float* dk = reinterpret_cast<const float*>(sm + Sh::Dks) + (t & (kTreeRing - 1)) * 64;
                const float* dv = reinterpret_cast<const float*>(sm + Sh::Dvs) + (t & (kTreeRing - 1)) * 64;
                gone = (key & 63) >= d.len;
                ks = gone ? 0.0f : dk[key & 63];
                const float vs = dv[key & 63] * kDraftedUnit;
                const float vtop = warp_max(fmaxf(lane < d.len ? dv[lane] : 0.0f, lane + 32 < d.len ? dv[lane + 32] : 0.0f)) * kDraftedUnit;
                const int ref = d.ref == -127 ? exponent_of(vtop) : d.ref;
                ve = (float)value_exponent(vs, ref);
                float f;
                f16_factor(vtop, kWeightBits + value_exponent(vtop, ref), f, un);
                vf = vs * f;
                un *= 1.0f / kDraftedUnit;
            }
            if (gone) vf = 0.0f;
            if (draft) {
                // scores of keys j and 64 + j together, through the weights' memory (tile t - 2's)
                float* x = reinterpret_cast<float*>(sm + Sh::P + t % PB * Sh::PParts * Sh::PPart) + part * QC * kTreeKeys;
#pragma unroll
                for (int c = 0; c < QC / 2; ++c) {
                    const float2 y = unpack2(s[c]);
                    x[2 * c * kTreeKeys + key] = y.x;
                    x[(2 * c + 1) * kTreeKeys + key] = y.y;
                }
                if (!meet()) break;
#pragma unroll
                for (int c = 0; c < QC / 2; ++c) s[c] = add2(s[c], pack2(x[2 * c * kTreeKeys + (key ^ 64)], x[(2 * c + 1) * kTreeKeys + (key ^ 64)]));
            }
            // scores in base 2 relative to h
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < QC / 2; x += 2) {
                const float4 un = *reinterpret_cast<const float4*>(unit + 2 * x), hh = *reinterpret_cast<const float4*>(bs + 2 * x);
                s[x] = fma2(s[x], mul2(pack2(un.x, un.y), pack2(ks, ks)), pack2(hh.x, hh.y));
                s[x + 1] = fma2(s[x + 1], mul2(pack2(un.z, un.w), pack2(ks, ks)), pack2(hh.z, hh.w));
            }
            if (draft) {
                const long long* seen = reinterpret_cast<const long long*>(sm + Sh::Seen) + it * NC + part * QC;
#pragma unroll
                for (int c = 0; c < QC / 2; ++c) {
                    float2 y = unpack2(s[c]);
                    if (gone || !(seen[2 * c] >> (key & 63) & 1)) y.x = -INFINITY;
                    if (gone || !(seen[2 * c + 1] >> (key & 63) & 1)) y.y = -INFINITY;
                    s[c] = pack2(y.x, y.y);
                }
            } else if (gone) {
#pragma unroll
                for (int c = 0; c < QC / 2; ++c) s[c] = pack2(-INFINITY, -INFINITY);
            }
#pragma unroll
            for (int x = 0; x < QC / 2; ++x) top = fmaxf(top, fmaxf(unpack2(s[x]).x, unpack2(s[x]).y));
            if (__any_sync(0xffffffffu, top + ve > kMoveBits) && lane == 0) moves[4 * (t & 1)] = t + 1;
            arrive_warp(&part_bar[part]);
            if (PB == 2 && !draft && begun > 1) fold(t - 2, u2, moved2);   // (by now its products are made)
            if (!ok || !wait_warp(&part_bar[part], met++ & 1, 20)) break;
            const bool moved = *reinterpret_cast<volatile int*>(&moves[4 * (t & 1)]) == t + 1 || __any_sync(0xffffffffu, unset);
            if (moved) {
                // the columns' largest, relative to h: lane c has column c
                float best = -INFINITY;
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    const float y0 = warp_max(unpack2(s[x]).x + ve), y1 = warp_max(unpack2(s[x]).y + ve);
                    if (lane == 2 * x) best = y0;
                    if (lane == 2 * x + 1) best = y1;
                }
                if (lane < QC) xm[(t & 1) * 16 * QC + quarter * QC + lane] = best;
                if (!meet()) break;
                float by = 0.0f;                               // how far h moves
                if (lane < QC) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) best = fmaxf(best, xm[(t & 1) * 16 * QC + q * QC + lane]);
                    by = rintf(unset ? (best > -INFINITY ? best : 0.0f) : fmaxf(best, 0.0f));
                    h += by;
                    bs[lane] = -h;
                    bk[(t & 1) * 16 * QC + lane] = unset ? 0.0f : exp2_fast(-0.5f * by);
                    bd[lane] = by;
                    unset = unset && !(best > -INFINITY);
                }
                __syncwarp();
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    const float2 dd = *reinterpret_cast<const float2*>(bd + 2 * x), bb = *reinterpret_cast<const float2*>(bk + (t & 1) * 16 * QC + 2 * x);
                    float2 y = unpack2(add2(s[x], pack2(-dd.x, -dd.y)));
                    // (scores so large that their sums with ve are roundings of it could end above what the weights hold)
                    if (y.x > kMoveBits - ve) y.x = kMoveBits - ve;
                    if (y.y > kMoveBits - ve) y.y = kMoveBits - ve;
                    s[x] = pack2(y.x, y.y);
                    l[x] = mul2(mul2(l[x], pack2(bb.x, bb.y)), pack2(bb.x, bb.y));      // (2^-by itself could leave f32's range)
                }
            }
            // probabilities, their sums, weights in the range of f16
            if (draft) {
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    const float2 y = unpack2(s[x]);
                    const float e0 = exp2_fast(y.x), e1 = exp2_fast(y.y);
                    if (key < 64) l[x] = add2(l[x], pack2(e0, e1));
                    // (what a column does not see weighs nothing, whatever its scale is)
                    s[x] = pack2(y.x == -INFINITY ? 0.0f : e0 * vf, y.y == -INFINITY ? 0.0f : e1 * vf);
                }
                arrive_warp(all_bar);                          // everybody has read the exchanged scores
                if (!wait_warp(all_bar, met_all++ & 1, 20)) break;
            } else {
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    const float2 y = unpack2(s[x]);
                    const f32x2 e = pack2(exp2_fast(y.x), exp2_fast(y.y));
                    l[x] = add2(l[x], e);
                    s[x] = mul2(e, pack2(vf, vf));
                }
            }
            if (PB == 1 && !draft && begun > 0) fold(t - 1, u1, moved1);
            if (!ok) break;
            unsigned char* pd = sm + Sh::P + t % PB * Sh::PParts * Sh::PPart + key * 128;
            uint32_t hi[QC / 2], lo[QC / 2];
#pragma unroll
            for (int x = 0; x < QC / 2; ++x) {
                const float2 y = unpack2(s[x]);
                split_f16(y.x, y.y, hi[x], lo[x]);
            }
            if constexpr (QC == 8) {
                *reinterpret_cast<uint4*>(pd + ((part ^ (key & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(pd + (((NC / 8 + part) ^ (key & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            } else {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    unsigned char* at = pd + (((2 * part + q) ^ (key & 7)) << 4);
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                    *reinterpret_cast<uint4*>(at + Sh::PPart) = make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
                }
            }
            fence_async_smem();
            arrive_warp(&pfull[t & 1]);
            u2 = u1; moved2 = moved1;
            u1 = un; moved1 = moved;
            if (flags & TREE_LAST) {
                if (PB == 2 && begun > 0) fold(t - 1, u2, moved2);
                fold(t, u1, moved1);
                if (!ok) break;
                // the item's sums over its keys, then its columns to memory
                // (the lanes halve the columns that they add up: lane x / (32 / QC) ends with column x)
                float z[QC];
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    const float2 y = unpack2(l[x]);
                    z[2 * x] = y.x; z[2 * x + 1] = y.y;
                }
                int keep = QC;
#pragma unroll
                for (int way = 16; way >= 1; way >>= 1) {
                    if (keep == 1) {
                        z[0] += __shfl_xor_sync(0xffffffffu, z[0], way);
                        continue;
                    }
                    keep /= 2;
                    const bool up = lane & way;
#pragma unroll
                    for (int x = 0; x < QC / 2; ++x) {
                        if (x >= keep) break;
                        const float give = __shfl_xor_sync(0xffffffffu, up ? z[x] : z[x + keep], way);
                        z[x] = (up ? z[x + keep] : z[x]) + give;
                    }
                }
                constexpr int Share = 32 / QC;
                if (lane % Share == 0) xl[quarter * QC + lane / Share] = z[0];
                if (!meet()) break;
                float sum = 0.0f;
                int sx = 0;
                if (lane < QC) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) sum += xl[q * QC + lane];
                    // (a split's sum is brought to [1, 2): h follows the values, and the joining takes powers of 2^h; where h
                    // is a whole number to which another can be added)
                    sx = sum > 0.0f && sum < INFINITY && fabsf(h) < 0x1p23f ? exponent_of(sum) : 0;
                    bd[lane] = d.nsplit > 1 ? __int_as_float((127 - sx) << 23) : sum == 0.0f ? 0.0f : fdiv(1.0f, sum);
                }
                __syncwarp();
                const int mine_col = part * QC + (lane & (QC - 1));
                float* mine_at = column_out(d, min(mine_col, d.cols - 1));
#pragma unroll
                for (int c = 0; c < OC; ++c) {
                    float* dst = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine_at), oc0 + c));
                    if (part * QC + oc0 + c >= d.cols) continue;
                    const float inv = bd[oc0 + c];
#pragma unroll
                    for (int mh = 0; mh < MH; ++mh) {
                        const float2 y = unpack2(o[mh][c / 2]);
                        if (oelem + 128 * mh < dh) dst[oelem + 128 * mh] = (c & 1 ? y.y : y.x) * inv;
                    }
                }
                if (d.nsplit > 1 && quarter == 0 && lane < QC && mine_col < d.cols) {
                    mine_at[dh] = unset ? -INFINITY : h + (float)sx;
                    mine_at[dh + 1] = sum * __int_as_float((127 - sx) << 23);
                }
            }
            arrive_warp(&tfree[t & (kTreeRing - 1)]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Sh::TmemCols) : "memory");
    }
    if (tid == 0 && *fail) set_err(p.err, B2_DEV_ERR_TIMEOUT);
}

// Joins the splits of each (row, head): grid (rows, heads * WPH / 8).
template <int WPH>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeAttnParams p) {
    __shared__ __align__(16) float so[8][256];
    __shared__ float sm[8][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y * (8 / WPH) + warp / WPH, row = blockIdx.x;
    after_previous();
    int n = 0;                                                 // the row's splits, the same for the whole CTA
    for (int base = 0; base < p.r.n_seq && n == 0; base += 32) {
        SeqRows q{0, 0, 0};
        if (base + lane < p.r.n_seq) q = seq_rows(p.r, base + lane);
        const unsigned m = __ballot_sync(0xffffffffu, row >= q.a && row < q.a + q.len);
        if (m) {
            const int src = __ffs(m) - 1, kv = __shfl_sync(0xffffffffu, q.kv, src), len = __shfl_sync(0xffffffffu, q.len, src);
            n = len > kTreeRows ? 1 : tree_splits(p.kc, min(kv, p.r.cap));
        }
    }
    if (n < 2) return;
    join_splits<WPH>(p.part + ((size_t)row * p.H + min(h, p.H - 1)) * p.nsplit * (p.c.dh + 4), n, p.c.dh, warp % WPH, warp, lane, so, sm,
                     h < p.H ? p.out + (size_t)row * p.ldo + (size_t)h * p.c.dh : nullptr);
}

}  // namespace b2
