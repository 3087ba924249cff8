// tree_attn.cuh — attention of drafted tokens over the paged 8-bit KV cache and over their own
// f32 keys and values (sm_100a).
//
// A sequence's drafted rows see all of its cached keys, so nothing is masked there: the
// columns (row, head) of a KV head meet every tile of 128 keys. Both products run on the 5th-
// generation tensor cores in f16 with the factors that are f32 held as two f16 each:
//   x f = hi + lo, f a power of two that brings the largest to [2^13, 2^14)
// which keeps 22 bits of every element down to 2^-28 of the largest, and at least 2^-39 of the
// largest of those below. The cached codes are exact in f16; drafted keys and values are two
// f16 too, as keys j and 64 + j of a tile of their own, so that all four products are made.
//   S^T [key][column] = K Q^T      hi and lo of Q one after another into the same sums
//   O^T [element][column] = V^T P  weights p x v_scale, hi and lo likewise
// Keys and elements lie on the TMEM lanes: a thread has one key of a few columns, whose scales
// are its own; the largest score of a column is found across the lanes. Each tile's output sums
// go to f32 registers, so that the tensor cores' sums stay short.
#pragma once
#include <cuda_fp16.h>

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
    int kc_log2, nsplit;     // a split: 2^kc_log2 cached keys, of which the last also has the
                             // drafted ones; nsplit: splits of cap keys
    float* part;             // [n_rows][H][nsplit][dh + 4]: o, m (base 2), l
    int* err;
};

__device__ __forceinline__ int tree_splits(int kc_log2, int keys) { return max((keys + (1 << kc_log2) - 1) >> kc_log2, 1); }

// Warps 0 .. 15, softmax: warp w reads TMEM lanes 32 (w % 4) .. + 31 and columns w / 4 of the
//   four parts of a tile's columns.
// Warps 16 .. 19: codes to f16 operands, the next tile's codes requested while this one's are
//   turned; an item's queries and drafted rows.
// Warp 20: issues the MMAs. Warp 21: finds the items (a sequence's columns of a KV head against
//   a split of its keys) and their tiles' blocks and scales, up to eight tiles ahead.
// A CTA a SM goes through its items with the pipeline running on from one to the next. Every
// wait is bounded; a warp whose wait ran out leaves its loop and sets the error word.
constexpr int kTreeSoftWarps = 16;
constexpr int kTreeConvWarps = 4;
constexpr int kTreeThreads = (kTreeSoftWarps + kTreeConvWarps + 2) * 32;
constexpr int kTreeRing = 8;
constexpr int kTreeKeys = 128;

enum { TREE_FIRST = 1, TREE_LAST = 2, TREE_DRAFT = 4, TREE_END = 8 };

struct TreeTile {
    int cell[8];             // block b of the tile in the pool (codes start at 16 dh times that; -1: none)
    float ks[8], vs[8];      // their scales (-1 and 0: none)
    int flags, item;
    int limit;               // keys of the tile
    int a, len, kvh;         // the item's rows and KV head,
    int col0, cols;          // its columns (row * G + head),
    int split, nsplit;
    int pad[2];
};

// DP: d_head rounded up to 64, 128 or 256; NC: columns of an item
template <int DP, int NC>
struct TreeShape {
    static constexpr int KS = DP == 64 ? 4 : DP == 128 ? 2 : 1;    // tiles of keys and values held
    static constexpr int Halves = DP / 64;                         // 128-byte parts of a row
    static constexpr int MH = DP == 256 ? 2 : 1;                   // 128 elements each of the output
    static constexpr int QC = NC / 4;                              // columns of a thread
    static constexpr int Tile = Halves * kTreeKeys * 128;          // [part][key][64 f16], swizzled
    static constexpr int QPart = Halves * NC * 128;                // [part][column][64 f16], swizzled
    static constexpr int PPart = kTreeKeys * 128;                  // [key][64 columns], swizzled
    static constexpr int K = 0;
    static constexpr int V = K + KS * Tile;
    static constexpr int Q = V + KS * Tile;                        // hi, lo
    static constexpr int P = Q + 2 * QPart;                        // hi, lo
    static constexpr int Ring = P + 2 * PPart;
    static constexpr int Unit = Ring + kTreeRing * (int)sizeof(TreeTile);       // [ring][NC] f32: of a column's scores
    static constexpr int Seen = Unit + kTreeRing * NC * 4;         // [ring][NC] words
    static constexpr int Dks = Seen + kTreeRing * NC * 8;          // [ring][64] scales of drafted keys
    static constexpr int Dvs = Dks + kTreeRing * 64 * 4;           // and values
    static constexpr int Xm = Dvs + kTreeRing * 64 * 4;            // [2][4 parts][4][QC] largest scores
    static constexpr int Xl = Xm + 2 * 16 * QC * 4;                // [4][4][QC] sums
    static constexpr int Bs = Xl + 16 * QC * 4;                    // [16 warps][QC]
    static constexpr int Bk = Bs + 16 * QC * 4;                    // [2][16][QC]
    static constexpr int Bars = Bk + 2 * 16 * QC * 4;
    static constexpr int NBars = 2 * kTreeRing + 4 * KS + 2 + 4 + 2 + 4 + 4 + 1 + 1;
    static constexpr int Bytes = Bars + NBars * 8 + 16;
    static constexpr int Alloc = Bytes + 1024;                     // operands start on 1024 bytes
    static constexpr int TmemS = 0, TmemO = 2 * NC;                // two buffers each
    static constexpr int TmemCols = 2 * NC + 2 * MH * NC <= 64 ? 64 : 256;
    static_assert(2 * NC + 2 * MH * NC <= 256 && Alloc <= 227 * 1024, "");
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

// two values as two f16 each: hi the nearest, lo what is left
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// the power of two that brings `top` (finite, >= 0) to [2^13, 2^14), and its reciprocal; tiny
// ones are brought as far as 2^126 does
__device__ __forceinline__ void f16_factor(float top, float& f, float& unit) {
    const int e = min(max(140 + 127 - (int)(__float_as_uint(top) >> 23), 1), 253);
    f = __int_as_float(e << 23);
    unit = __int_as_float((254 - e) << 23);
}

__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

// A row of DP f32 elements (16 lanes, lane l16 the elements 4 l16 + 64 i ..) as hi and lo at
// hi_at(i, unit) and lo_at: the 16-byte unit of part i. Returns the scale of its values: NaN for a
// row that is not finite (its elements are zeros then, so that they harm no one else).
template <int DP, typename At>
__device__ __forceinline__ float put_row_f16(const float* src, bool live, int dh, int l16, At hi_at, At lo_at) {
    float4 x[DP / 64];
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        const int d = 4 * l16 + 64 * i;
        x[i] = live && d < dh ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        bad |= x[i].x != x[i].x || x[i].y != x[i].y || x[i].z != x[i].z || x[i].w != x[i].w;
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float f, unit;
    f16_factor(top, f, unit);
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
__global__ void __launch_bounds__(kTreeThreads, 1) tree_attn_kernel(const __grid_constant__ TreeAttnParams p) {
    using Sh = TreeShape<DP, NC>;
    constexpr int KS = Sh::KS, QC = Sh::QC, MH = Sh::MH;
    extern __shared__ unsigned char ta_raw[];
    unsigned char* sm = ta_raw + ((1024u - (smem_u32(ta_raw) & 1023u)) & 1023u);
    TreeTile* ring = reinterpret_cast<TreeTile*>(sm + Sh::Ring);
    uint64_t* tready = reinterpret_cast<uint64_t*>(sm + Sh::Bars);     // [ring] a tile is described
    uint64_t* tfree = tready + kTreeRing;                              // [ring] and not needed any more
    uint64_t* kfull = tfree + kTreeRing;                               // [KS] keys written
    uint64_t* kempty = kfull + KS;                                     // [KS] their scores are made
    uint64_t* vfull = kempty + KS;
    uint64_t* vempty = vfull + KS;
    uint64_t* qfull = vempty + KS;                                     // an item's queries written
    uint64_t* qfree = qfull + 1;                                       // its last scores made
    uint64_t* sfull = qfree + 1;                                       // [2] scores in TMEM
    uint64_t* sfree = sfull + 2;                                       // [2] read
    uint64_t* pfull = sfree + 2;                                       // weights written
    uint64_t* pfree = pfull + 1;                                       // their products made
    uint64_t* ofull = pfree + 1;                                       // [2] output sums in TMEM
    uint64_t* ofree = ofull + 2;                                       // [2] read
    uint64_t* part_bar = ofree + 2;                                    // [4] the warps of a column part meet
    uint64_t* all_bar = part_bar + 4;                                  // all softmax warps meet
    uint64_t* done = all_bar + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int dh = p.c.dh;
    constexpr int kMmaWarp = kTreeSoftWarps + kTreeConvWarps, kPlanWarp = kMmaWarp + 1;

    after_previous();
    if (tid == 0) {
        for (int i = 0; i < kTreeRing; ++i) { mbar_init(&tready[i], 1); mbar_init(&tfree[i], kTreeSoftWarps + kTreeConvWarps + 1); }
        for (int i = 0; i < KS; ++i) {
            mbar_init(&kfull[i], kTreeConvWarps * 32); mbar_init(&kempty[i], 1);
            mbar_init(&vfull[i], kTreeConvWarps * 32); mbar_init(&vempty[i], 1);
        }
        mbar_init(qfull, kTreeConvWarps * 32); mbar_init(qfree, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sfull[i], 2); mbar_init(&sfree[i], kTreeSoftWarps);
            mbar_init(&ofull[i], 1); mbar_init(&ofree[i], kTreeSoftWarps);
        }
        mbar_init(pfull, kTreeSoftWarps); mbar_init(pfree, 1);
        for (int i = 0; i < 4; ++i) mbar_init(&part_bar[i], 4);
        mbar_init(all_bar, kTreeSoftWarps); mbar_init(done, 1);
        fence_mbar_init();
        *fail = 0;
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
        int t = 0, base = 0;
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
                        cnt = (unsigned)(((q.len * p.G + NC - 1) / NC) * p.c.KVH * tree_splits(p.kc_log2, min(q.kv, p.r.cap)));
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
            const int ctiles = (len * p.G + NC - 1) / NC, nsplit = tree_splits(p.kc_log2, kv);
            const int ct = (int)(idx % (unsigned)ctiles), rest = (int)(idx / (unsigned)ctiles), kvh = rest % p.c.KVH, split = rest / p.c.KVH;
            const int j0 = split << p.kc_log2, jend = min(kv, j0 + (1 << p.kc_log2));
            const int ntiles = (max(jend - j0, 0) + kTreeKeys - 1) / kTreeKeys, all = ntiles + (split == nsplit - 1);
            for (int i0 = 0; i0 < all && ok; i0 += 4) {
                const int i = i0 + group, j = j0 + i * kTreeKeys + 16 * b, cnt = min(all - i0, 4);
                int cell = -1;
                float ks = -1.0f, vs = 0.0f;
                if (i < ntiles && j < jend) {
                    const int page = page_of(p.c, p.r, s, j);
                    if (page < 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
                    else {
                        cell = (page * p.c.KVH + kvh) * (psz >> 4) + ((j & (psz - 1)) >> 4);
                        ks = p.c.ks[cell];
                        vs = p.c.vs[cell];
                    }
                }
                for (int u = 0; u < cnt && ok; ++u)
                    if (t + u >= kTreeRing) ok = wait_warp(&tfree[(t + u) & (kTreeRing - 1)], ring_parity(t + u) ^ 1, 100);
                if (!ok) break;
                if (group < cnt) {
                    TreeTile& d = ring[(t + group) & (kTreeRing - 1)];
                    d.cell[b] = cell; d.ks[b] = ks; d.vs[b] = vs;
                    if (b == 0) {
                        d.flags = (i == 0 ? TREE_FIRST : 0) | (i == all - 1 ? TREE_LAST : 0) | (i == ntiles ? TREE_DRAFT : 0);
                        d.item = n; d.limit = jend - (j0 + i * kTreeKeys);
                        d.a = a; d.len = len; d.kvh = kvh; d.col0 = ct * NC; d.cols = min(len * p.G - ct * NC, NC);
                        d.split = split; d.nsplit = nsplit;
                    }
                }
                __syncwarp();
                if (lane < cnt) mbar_arrive(&tready[(t + lane) & (kTreeRing - 1)]);
                t += cnt;
            }
        }
    } else if (warp == kMmaWarp) {
        // ---- MMAs (one lane)
        if (lane == 0) {
            const uint32_t base = smem_u32(sm);
            const uint32_t ids = umma_idesc_f16(NC, false, false), ido = umma_idesc_f16(NC, true, true);
            bool ok = true;
            int items = 0;
            auto scores = [&](int t, int flags) {
                const int slot = t % KS, use = t / KS;
                ok = ok && wait(&kfull[slot], use & 1, 20);
                if (ok && (flags & TREE_FIRST)) ok = wait(qfull, items & 1, 20);
                if (ok && t > 1) ok = wait(&sfree[t & 1], ((t >> 1) - 1) & 1, 20);
                if (!ok) return;
                tc_fence_after();
                const uint32_t kb = base + Sh::K + slot * Sh::Tile, qb = base + Sh::Q;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int h = 0; h < Sh::Halves; ++h)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16(tmem + Sh::TmemS + (t & 1) * NC, umma_desc_sw128(kb + h * kTreeKeys * 128 + 32 * k),
                                     umma_desc_sw128(qb + e * Sh::QPart + h * NC * 128 + 32 * k), ids, e + h + k > 0 ? 1u : 0u);
                umma_commit(&kempty[slot]);
                if (flags & TREE_LAST) {
                    umma_commit(qfree);
                    ++items;
                }
                umma_commit(&sfull[t & 1]);
                mbar_arrive(&sfull[t & 1]);                    // passes on what the others wrote: units, scales
            };
            auto output = [&](int t) {
                const int slot = t % KS, use = t / KS;
                ok = ok && wait(pfull, t & 1, 20) && wait(&vfull[slot], use & 1, 20);
                if (ok && t > 1) ok = wait(&ofree[t & 1], ((t >> 1) - 1) & 1, 20);
                if (!ok) return;
                tc_fence_after();
                const uint32_t vb = base + Sh::V + slot * Sh::Tile, pb = base + Sh::P;
#pragma unroll
                for (int mh = 0; mh < MH; ++mh)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int k = 0; k < kTreeKeys / 16; ++k)      // (d_head 64: lanes 64 .. 127 repeat the others)
                            umma_f16(tmem + Sh::TmemO + ((t & 1) * MH + mh) * NC,
                                     umma_desc_sw128_mn(vb + mh * 2 * kTreeKeys * 128 + k * 2048, Sh::Halves > 1 ? kTreeKeys * 128 : 0),
                                     umma_desc_sw128_mn(pb + e * Sh::PPart + k * 2048, 0), ido, e + k > 0 ? 1u : 0u);
                umma_commit(&vempty[slot]);
                umma_commit(pfree);
                umma_commit(&ofull[t & 1]);
            };
            // the flags of tile t; its description is not needed after that
            auto flags_of = [&](int t) {
                ok = ok && wait(&tready[t & (kTreeRing - 1)], ring_parity(t), 20);
                const int f = ok ? ring[t & (kTreeRing - 1)].flags : TREE_END;
                if (ok) mbar_arrive(&tfree[t & (kTreeRing - 1)]);
                return f;
            };
            int flags = flags_of(0);
            if (!(flags & TREE_END)) scores(0, flags);
            for (int t = 0; ok && !(flags & TREE_END); ++t) {
                flags = flags_of(t + 1);
                // the next tile's scores go first, except those of another item, whose queries
                // wait for this one's, and drafted ones where they wait for the only values' place
                const bool ahead = !(flags & (TREE_END | TREE_FIRST)) && !(KS == 1 && (flags & TREE_DRAFT));
                if (ahead) scores(t + 1, flags);
                output(t);
                if (!ahead && !(flags & TREE_END)) scores(t + 1, flags);
            }
            umma_commit(done);                                 // also after a wait that ran out: no MMA may be
            if (!mbar_wait_bounded(done, 0)) *fail = 1;        // under way when its memory is given up
        }
    } else if (warp >= kTreeSoftWarps) {
        // ---- operands
        constexpr int Chunks = DP / 16;                        // 16 codes each of a row
        constexpr int Units = kTreeKeys * Chunks / (kTreeConvWarps * 32), UR = Units < 8 ? Units : 8, Rounds = Units / UR;
        const int ct = tid - kTreeSoftWarps * 32, chunk = ct % Chunks, key0 = ct / Chunks;
        constexpr int KeyStep = kTreeConvWarps * 32 / Chunks;
        uint4 kr[UR], vr[UR];
        auto fetch = [&](const TreeTile& d, const int8_t* codes, int round, uint4 (&r)[UR]) {
#pragma unroll
            for (int x = 0; x < UR; ++x) {
                const int key = key0 + (round * UR + x) * KeyStep, cell = d.cell[key >> 4];
                r[x] = cell >= 0 && 16 * chunk < dh ? load16(codes + ((size_t)cell * kKvBlock + (key & 15)) * dh + 16 * chunk)
                                                    : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        auto put = [&](unsigned char* tile, int round, const uint4 (&r)[UR]) {
            unsigned char* part = tile + (chunk >> 2) * kTreeKeys * 128;
            const int u0 = 2 * (chunk & 3), turn = (chunk >> 2) & 1;      // (parts in turn: no bank conflicts)
#pragma unroll
            for (int x = 0; x < UR; ++x) {
                const int key = key0 + (round * UR + x) * KeyStep;
                const uint4 lo = codes_f16(r[x].x, r[x].y), hi = codes_f16(r[x].z, r[x].w);
                unsigned char* row = part + key * 128;
                *reinterpret_cast<uint4*>(row + (((u0 + turn) ^ (key & 7)) << 4)) = turn ? hi : lo;
                *reinterpret_cast<uint4*>(row + (((u0 + 1 - turn) ^ (key & 7)) << 4)) = turn ? lo : hi;
            }
        };
        // drafted rows: key j and 64 + j of the tile (zeros past the last)
        auto put_drafted = [&](unsigned char* tile, const TreeTile& d, const float* src, long long ld, float* scales) {
            for (int r0 = 0; r0 < 64; r0 += kTreeConvWarps * 2) {
                const int j = r0 + (ct >> 4);
                auto at = [&](int row) {
                    return [=](int i, int u) { return tile + i * kTreeKeys * 128 + row * 128 + ((u ^ (row & 7)) << 4); };
                };
                const float unit = put_row_f16<DP>(src + (size_t)(d.a + min(j, d.len - 1)) * ld + (size_t)d.kvh * dh, j < d.len, dh, ct & 15,
                                                   at(j), at(64 + j));
                if ((ct & 15) == 0) scales[j] = unit;
            }
        };
        bool ok = wait_warp(&tready[0], 0, 20);
        if (ok && !(ring[0].flags & (TREE_DRAFT | TREE_END))) {
            fetch(ring[0], p.c.k, 0, kr);
            fetch(ring[0], p.c.v, 0, vr);
        }
        for (int t = 0; ok; ++t) {
            const TreeTile& d = ring[t & (kTreeRing - 1)];
            if (d.flags & TREE_END) break;
            const int slot = t % KS, use = t / KS;
            const bool draft = d.flags & TREE_DRAFT;
            if (d.flags & TREE_FIRST) {
                if (d.item > 0) ok = wait_warp(qfree, (d.item - 1) & 1, 50);
                if (!ok) break;
                const int it = d.item & (kTreeRing - 1);
                float* unit = reinterpret_cast<float*>(sm + Sh::Unit) + it * NC;
                long long* seen = reinterpret_cast<long long*>(sm + Sh::Seen) + it * NC;
#pragma unroll 2
                for (int c0 = 0; c0 < NC; c0 += kTreeConvWarps * 2) {
                    const int c = c0 + (ct >> 4), cc = d.col0 + min(c, d.cols - 1), tok = cc / p.G;
                    auto at = [&](int e) {
                        return [=](int i, int u) { return sm + Sh::Q + e * Sh::QPart + i * NC * 128 + c * 128 + ((u ^ (c & 7)) << 4); };
                    };
                    const float un = put_row_f16<DP>(p.q + (size_t)(d.a + tok) * p.ldq + (size_t)(d.kvh * p.G + cc - tok * p.G) * dh, c < d.cols,
                                                     dh, ct & 15, at(0), at(1));
                    if ((ct & 15) == 0) {
                        unit[c] = un * 1.4426950408889634f;            // log2 e
                        seen[c] = c < d.cols ? p.seen[d.a + tok] : 0;
                    }
                }
                fence_async_smem();
                mbar_arrive(qfull);
            }
            ok = ok && wait_warp(&tready[(t + 1) & (kTreeRing - 1)], ring_parity(t + 1), 20);
            if (!ok) break;
            const TreeTile& nx = ring[(t + 1) & (kTreeRing - 1)];
            const bool more = !(nx.flags & (TREE_DRAFT | TREE_END));
            if (t >= KS) ok = wait_warp(&kempty[slot], (use - 1) & 1, 50);
            if (!ok) break;
            unsigned char* kd = sm + Sh::K + slot * Sh::Tile;
            if (draft) {
                put_drafted(kd, d, p.k, p.ldk, reinterpret_cast<float*>(sm + Sh::Dks) + (t & (kTreeRing - 1)) * 64);
            } else {
#pragma unroll
                for (int r = 0; r < Rounds; ++r) {
                    if (r > 0) fetch(d, p.c.k, r, kr);
                    put(kd, r, kr);
                }
            }
            if (more) fetch(nx, p.c.k, 0, kr);
            unsigned char* vd = sm + Sh::V + slot * Sh::Tile;
            float* dvs = reinterpret_cast<float*>(sm + Sh::Dvs) + (t & (kTreeRing - 1)) * 64;
            if (draft) {                                       // both before the scores: the softmax wants all scales
                if (t >= KS) ok = wait_warp(&vempty[slot], (use - 1) & 1, 50);
                if (!ok) break;
                put_drafted(vd, d, p.v, p.ldv, dvs);
                fence_async_smem();
                mbar_arrive(&kfull[slot]);
            } else {
                fence_async_smem();
                mbar_arrive(&kfull[slot]);
                if (t >= KS) ok = wait_warp(&vempty[slot], (use - 1) & 1, 50);
                if (!ok) break;
#pragma unroll
                for (int r = 0; r < Rounds; ++r) {
                    if (r > 0) fetch(d, p.c.v, r, vr);
                    put(vd, r, vr);
                }
                fence_async_smem();
            }
            mbar_arrive(&vfull[slot]);
            if (more) fetch(nx, p.c.v, 0, vr);
            arrive_warp(&tfree[t & (kTreeRing - 1)]);
        }
    } else {
        // ---- softmax and output
        const int quarter = warp & 3, part = warp >> 2, key = 32 * quarter + lane;
        const uint32_t trow = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(part * QC);
        float* bs = reinterpret_cast<float*>(sm + Sh::Bs) + warp * QC;
        float* bk = reinterpret_cast<float*>(sm + Sh::Bk) + warp * QC;
        float* xm = reinterpret_cast<float*>(sm + Sh::Xm) + part * 4 * QC;
        float* xl = reinterpret_cast<float*>(sm + Sh::Xl) + part * 4 * QC;
        int met = 0, met_all = 0;                              // how often the part's warps, all of them have met
        bool ok = true;
        auto meet = [&]() {
            arrive_warp(&part_bar[part]);
            ok = wait_warp(&part_bar[part], met++ & 1, 20);
            return ok;
        };
        auto read_cols = [&](uint32_t at, uint32_t (&r)[QC]) {
            if constexpr (QC == 16) tmem_ld16(at, r);
            else if constexpr (QC == 8) tmem_ld8(at, r);
            else tmem_ld4(at, r);
        };
        float m = -INFINITY;                                   // of column `lane`
        f32x2 l[QC / 2], o[MH][QC / 2];
        float u = 0.0f;                                        // of the tile whose output is pending
        // output sums of tile t
        auto fold = [&](int t) {
            ok = ok && wait_warp(&ofull[t & 1], (t >> 1) & 1, 20);
            if (!ok) return;
            tc_fence_after();
            uint32_t c[MH][QC];
#pragma unroll
            for (int mh = 0; mh < MH; ++mh) read_cols(trow + Sh::TmemO + ((t & 1) * MH + mh) * NC, c[mh]);
            tmem_wait_ld();
            tc_fence_before();
            arrive_warp(&ofree[t & 1]);
            const float* back = bk + (t & 1) * 16 * QC;
#pragma unroll
            for (int x = 0; x < QC / 2; ++x) {
                const float2 bb = *reinterpret_cast<const float2*>(back + 2 * x);
#pragma unroll
                for (int mh = 0; mh < MH; ++mh)
                    o[mh][x] = fma2(pack2(__uint_as_float(c[mh][2 * x]), __uint_as_float(c[mh][2 * x + 1])), pack2(u, u),
                                    mul2(o[mh][x], pack2(bb.x, bb.y)));
            }
        };
        for (int t = 0; ok; ++t) {
            if (!wait_warp(&tready[t & (kTreeRing - 1)], ring_parity(t), 20)) break;
            const TreeTile& d = ring[t & (kTreeRing - 1)];
            const int flags = d.flags;
            if (flags & TREE_END) break;
            const bool draft = flags & TREE_DRAFT;
            if (flags & TREE_FIRST) {
                m = -INFINITY;
#pragma unroll
                for (int x = 0; x < QC / 2; ++x) {
                    l[x] = 0ull;
#pragma unroll
                    for (int mh = 0; mh < MH; ++mh) o[mh][x] = 0ull;
                }
            }
            const int it = d.item & (kTreeRing - 1);
            const float* unit = reinterpret_cast<const float*>(sm + Sh::Unit) + it * NC + part * QC;
            if (!wait_warp(&sfull[t & 1], (t >> 1) & 1, 20)) break;
            tc_fence_after();
            uint32_t raw[QC];
            read_cols(trow + Sh::TmemS + (t & 1) * NC, raw);
            // this key's scales, and the largest value scale of the tile
            float ks, vs, vtop = 0.0f;
            bool gone;
            if (!draft) {
                ks = d.ks[key >> 4];
                vs = d.vs[key >> 4];
                gone = ks < 0.0f || key >= d.limit;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(&d.vs[i]);
                    vtop = fmaxf(vtop, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
                }
            } else {
                const float* dk = reinterpret_cast<const float*>(sm + Sh::Dks) + (t & (kTreeRing - 1)) * 64;
                const float* dv = reinterpret_cast<const float*>(sm + Sh::Dvs) + (t & (kTreeRing - 1)) * 64;
                ks = dk[key & 63];
                vs = dv[key & 63];
                gone = (key & 63) >= d.len;
                for (int i = 0; i < d.len; ++i) vtop = fmaxf(vtop, dv[i]);
            }
            if (gone) vs = 0.0f;
            tmem_wait_ld();
            tc_fence_before();
            arrive_warp(&sfree[t & 1]);
            if (draft) {
                // scores of keys j and 64 + j together, through the weights' memory
                if (t > 0 && !wait_warp(pfree, (t - 1) & 1, 20)) break;
                float* x = reinterpret_cast<float*>(sm + Sh::P) + part * QC * kTreeKeys;
#pragma unroll
                for (int c = 0; c < QC; ++c) x[c * kTreeKeys + key] = __uint_as_float(raw[c]);
                if (!meet()) break;
#pragma unroll
                for (int c = 0; c < QC; ++c) raw[c] = __float_as_uint(__uint_as_float(raw[c]) + x[c * kTreeKeys + (key ^ 64)]);
                asm volatile("" ::: "memory");
            }
            float s[QC];
#pragma unroll
            for (int x = 0; x < QC; x += 2) {
                const float2 un = *reinterpret_cast<const float2*>(unit + x);
                const float2 y = unpack2(mul2(pack2(__uint_as_float(raw[x]), __uint_as_float(raw[x + 1])),
                                              mul2(pack2(un.x, un.y), pack2(ks, ks))));
                s[x] = gone ? -INFINITY : y.x;
                s[x + 1] = gone ? -INFINITY : y.y;
            }
            if (draft) {
                const long long* seen = reinterpret_cast<const long long*>(sm + Sh::Seen) + it * NC + part * QC;
#pragma unroll
                for (int c = 0; c < QC; ++c)
                    if (!(seen[c] >> (key & 63) & 1)) s[c] = -INFINITY;
            }
            // the columns' largest scores: lane c has column c
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                const float y = warp_max(s[c]);
                if (lane == c) top = y;
            }
            if (lane < QC) xm[(t & 1) * 16 * QC + quarter * QC + lane] = top;
            if (!meet()) break;
            if (lane < QC) {
#pragma unroll
                for (int q = 0; q < 4; ++q) top = fmaxf(top, xm[(t & 1) * 16 * QC + q * QC + lane]);
                top = fmaxf(top, m);
                const float h = top == -INFINITY ? 0.0f : top;
                bs[lane] = h;
                bk[(t & 1) * 16 * QC + lane] = exp2_fast(m - h);
                m = top;
            }
            __syncwarp();
            // probabilities, their sums, weights in the range of f16
            float f, un;
            f16_factor(vtop, f, un);
            const float vf = vs * f;
            const bool count = !draft || key < 64;
#pragma unroll
            for (int x = 0; x < QC; x += 2) {
                const float2 h = *reinterpret_cast<const float2*>(bs + x), bb = *reinterpret_cast<const float2*>(bk + (t & 1) * 16 * QC + x);
                const float e0 = exp2_fast(s[x] - h.x), e1 = exp2_fast(s[x + 1] - h.y);
                l[x / 2] = fma2(l[x / 2], pack2(bb.x, bb.y), count ? pack2(e0, e1) : 0ull);
                // (what a column does not see weighs nothing, whatever its scale is)
                s[x] = draft && s[x] == -INFINITY ? 0.0f : e0 * vf;
                s[x + 1] = draft && s[x + 1] == -INFINITY ? 0.0f : e1 * vf;
            }
            if (!draft && t > 0 && !wait_warp(pfree, (t - 1) & 1, 20)) break;
            if (draft) {                                       // everybody has read the exchanged scores
                arrive_warp(all_bar);
                if (!wait_warp(all_bar, met_all++ & 1, 20)) break;
            }
            unsigned char* pd = sm + Sh::P + key * 128;
            uint32_t hi[QC / 2], lo[QC / 2];
#pragma unroll
            for (int x = 0; x < QC / 2; ++x) split_f16(s[2 * x], s[2 * x + 1], hi[x], lo[x]);
            if constexpr (QC == 4) {
                unsigned char* at = pd + (((part >> 1) ^ (key & 7)) << 4) + 8 * (part & 1);
                *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(at + Sh::PPart) = make_uint2(lo[0], lo[1]);
            } else {
#pragma unroll
                for (int q = 0; q < QC / 8; ++q) {
                    unsigned char* at = pd + (((part * (QC / 8) + q) ^ (key & 7)) << 4);
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                    *reinterpret_cast<uint4*>(at + Sh::PPart) = make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
                }
            }
            fence_async_smem();
            arrive_warp(pfull);
            if (!(flags & TREE_FIRST)) fold(t - 1);
            u = un;
            if (flags & TREE_LAST) {
                fold(t);
                if (!ok) break;
                // the item's sums over its keys, then its columns to memory
                float mine = 0.0f;
#pragma unroll
                for (int c = 0; c < QC; ++c) {
                    const float2 y = unpack2(l[c / 2]);
                    const float z = butterfly32(c & 1 ? y.y : y.x);
                    if (lane == c) mine = z;
                }
                if (lane < QC) xl[quarter * QC + lane] = mine;
                if (!meet()) break;
                float sum = 0.0f;
                if (lane < QC) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) sum += xl[q * QC + lane];
                    bs[lane] = d.nsplit > 1 ? 1.0f : sum == 0.0f ? 0.0f : fdiv(1.0f, sum);
                }
                __syncwarp();
                for (int c = 0; c < QC; ++c) {
                    const int col = part * QC + c;
                    if (col >= d.cols) break;
                    const int cc = d.col0 + col, tok = cc / p.G, row = d.a + tok, h = d.kvh * p.G + cc - tok * p.G;
                    float* dst = d.nsplit > 1 ? p.part + (((size_t)row * p.H + h) * p.nsplit + d.split) * (dh + 4)
                                              : p.out + (size_t)row * p.ldo + (size_t)h * dh;
                    const float inv = bs[c];
#pragma unroll
                    for (int mh = 0; mh < MH; ++mh) {
                        float y = 0.0f;                        // (registers are not indexed)
#pragma unroll
                        for (int x = 0; x < QC / 2; ++x) {
                            const float2 z = unpack2(o[mh][x]);
                            if (c == 2 * x) y = z.x;
                            if (c == 2 * x + 1) y = z.y;
                        }
                        if (key + 128 * mh < dh) dst[key + 128 * mh] = y * inv;
                    }
                    if (d.nsplit > 1 && quarter == 0 && lane == c) { dst[dh] = m; dst[dh + 1] = sum; }
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
            n = len > kTreeRows ? 1 : tree_splits(p.kc_log2, min(kv, p.r.cap));
        }
    }
    if (n < 2) return;
    join_splits<WPH>(p.part + ((size_t)row * p.H + min(h, p.H - 1)) * p.nsplit * (p.c.dh + 4), n, p.c.dh, warp % WPH, warp, lane, so, sm,
                     h < p.H ? p.out + (size_t)row * p.ldo + (size_t)h * p.c.dh : nullptr);
}

}  // namespace b2
