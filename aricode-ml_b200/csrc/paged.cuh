// paged.cuh — the paged 8-bit KV cache: norms and rotation of queries and keys,
// appending rows, reading rows back, attention (sm_100a).
//
// Cache: pages of `page` tokens; per page and KV head, K and V are int8 rows
// [page][dh] with one f32 scale per block of 16 tokens. A call's rows are ragged:
// sequence s has rows row_start[s] .. row_start[s + 1] - 1, the last of its
// kv_len[s] keys, so row i of it stands at position kv_len[s] - len + i. Lengths,
// starts and pages are read on the device only (a captured launch replays with new
// ones); every value is checked before it becomes an address.
#pragma once
#include "kernels.cuh"

namespace b2 {

constexpr int kKvBlock = 16;           // tokens that share a scale

struct PagedKv {
    int8_t* k;               // [n_pages][KVH][page][dh]
    int8_t* v;
    float* ks;               // [n_pages][KVH][page / 16]
    float* vs;
    int n_pages, page_log2, KVH, dh;
};

struct PagedRows {
    const int* row_start;    // [n_seq + 1]
    const int* kv_len;       // [n_seq]
    const int* table;        // [n_seq][max_pages]
    int n_seq, max_pages, n_rows;
    int cap;                 // positions a sequence can hold: min(max_keys, max_pages * page)
};

// one sequence's rows: a .. a + len - 1, at positions pos0 .. pos0 + len - 1
// (negative ones stand nowhere), keys 0 .. min(kv, cap) - 1
struct SeqRows {
    int a, len, kv;
    __device__ __forceinline__ int pos0() const { return kv - len; }
};

__device__ __forceinline__ SeqRows seq_rows(const PagedRows& r, int s) {
    SeqRows q;
    q.a = min(max(__ldg(r.row_start + s), 0), r.n_rows);
    q.len = min(max(__ldg(r.row_start + s + 1), q.a), r.n_rows) - q.a;
    q.kv = max(__ldg(r.kv_len + s), 0);
    return q;
}

// page of position pos of sequence s, or -1
__device__ __forceinline__ int page_of(const PagedKv& c, const PagedRows& r, int s, int pos) {
    const int id = __ldg(r.table + (size_t)s * r.max_pages + (pos >> c.page_log2));
    return (unsigned)id < (unsigned)c.n_pages ? id : -1;
}

// A run: the rows of one sequence that lie in one block of 16 tokens.
struct BlockRun {
    int s;          // sequence (-1: none)
    int row, n;     // its rows row .. row + n - 1 (1 <= n <= 16)
    int pos;        // position of the first one
};

// Run number `item` of the call, found by one warp: lanes count the runs of 32
// sequences at a time. `most` = runs the grid covers (more than that only if the
// row ranges overlap).
__device__ __forceinline__ BlockRun find_run(const PagedRows& r, int item, int most, int* err, int lane) {
    BlockRun out{-1, 0, 0, 0};
    int before = 0;
    bool found = false;
    for (int base = 0; base < r.n_seq; base += 32) {
        const int s = base + lane;
        int nb = 0, first = 0;
        SeqRows q{0, 0, 0};
        if (s < r.n_seq) {
            q = seq_rows(r, s);
            first = max(q.pos0(), 0);
            const int last = min(q.kv, r.cap) - 1;
            if (q.len > 0 && q.kv > r.cap && item == 0) set_err(err, B2_DEV_ERR_KV_OVERFLOW);
            if (q.len > 0 && last >= first) nb = last / kKvBlock - first / kKvBlock + 1;
        }
        int incl = nb;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const int total = __shfl_sync(0xffffffffu, incl, 31);
        if (!found && item < before + total) {
            const unsigned m = __ballot_sync(0xffffffffu, before + incl > item);
            const int src = __ffs(m) - 1;
            const int idx = item - before - (incl - nb);          // run within the sequence (lane src)
            const int b0 = first / kKvBlock + idx;
            const int p0 = max(b0 * kKvBlock, first);
            const int p1 = min(min(b0 * kKvBlock + kKvBlock, q.kv), r.cap);
            out.s = __shfl_sync(0xffffffffu, s, src);
            out.row = __shfl_sync(0xffffffffu, q.a + (p0 - q.pos0()), src);
            out.n = __shfl_sync(0xffffffffu, p1 - p0, src);
            out.pos = __shfl_sync(0xffffffffu, p0, src);
            found = true;
            if (item != 0) return out;                            // item 0 also checks the rest
        }
        before += total;
    }
    if (item == 0 && before > most && lane == 0) set_err(err, B2_DEV_ERR_BAD_ROWS);
    return out;
}

// ------------------------------------------------------------------ norm + rotation
// Head vectors in registers: LPH lanes hold a vector, VPL float4s each (lane l of
// the group the elements 4 l + 128 i ..), so dh <= 4 LPH VPL.
template <int LPH, int VPL>
__device__ __forceinline__ void head_norm(float4 (&x)[VPL], const float4 (&g)[VPL], int dh, float eps) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        a = fadd(a, fadd(fadd(fmul(x[i].x, x[i].x), fmul(x[i].y, x[i].y)),
                         fadd(fmul(x[i].z, x[i].z), fmul(x[i].w, x[i].w))));
#pragma unroll
    for (int o = LPH / 2; o >= 1; o >>= 1) a = fadd(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float r = fdiv(1.0f, __fsqrt_rn(fadd(fdiv(a, (float)dh), eps)));
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        x[i].x = fmul(fmul(x[i].x, r), g[i].x);
        x[i].y = fmul(fmul(x[i].y, r), g[i].y);
        x[i].z = fmul(fmul(x[i].z, r), g[i].z);
        x[i].w = fmul(fmul(x[i].w, r), g[i].w);
    }
}

// two neighbouring pairs by (cos, sin, cos, sin): b2_rope_apply's arithmetic
__device__ __forceinline__ float4 rotate4(const float4& x, const float4& t) {
    float4 y;
    y.x = fsub(fmul(x.x, t.x), fmul(x.y, t.y));
    y.y = fadd(fmul(x.x, t.y), fmul(x.y, t.x));
    y.z = fsub(fmul(x.z, t.z), fmul(x.w, t.w));
    y.w = fadd(fmul(x.z, t.w), fmul(x.w, t.z));
    return y;
}

struct NormRopeParams {
    const float* q;          // [n_rows][ldq], H heads side by side
    const float* k;          // [n_rows][ldk]
    float* qo;
    float* ko;
    long long ldq, ldk, ldqo, ldko;
    const float* gq;         // [dh] or nullptr: no norm
    const float* gk;
    float eps, q_scale;
    const float* table;      // [table_rows][dh] (cos, sin) pairs or nullptr: no rotation
    int table_rows;
    const int* pos;          // [n_rows]; negative: the row is left alone
    int n_rows, H, KVH, dh;
    int* err;
};

// HPU vectors of one row through norm, rotation and scale, all loads first. `h0`
// the first of them in the row's list (queries, then keys); `live`: the group has
// work (every lane of the warp runs along for the shuffles).
template <int LPH, int VPL, int HPU>
__device__ __forceinline__ void norm_rope_heads(const NormRopeParams& p, int row, int h0, int gl, bool live,
                                                int pos) {
    const int NH = p.H + p.KVH;
    float4 x[HPU][VPL];
#pragma unroll
    for (int u = 0; u < HPU; ++u) {
        const int h = h0 + u;
        const float* src = h < p.H ? p.q + (size_t)row * p.ldq + (size_t)h * p.dh
                                   : p.k + (size_t)row * p.ldk + (size_t)(h - p.H) * p.dh;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int d = 4 * (gl + LPH * i);
            x[u][i] = (live && h < NH && d < p.dh) ? *reinterpret_cast<const float4*>(src + d)
                                                   : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    float4 t[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int d = 4 * (gl + LPH * i);
        t[i] = (live && p.table && d < p.dh)
                   ? __ldg(reinterpret_cast<const float4*>(p.table + (size_t)pos * p.dh + d))
                   : make_float4(1.f, 0.f, 1.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < HPU; ++u) {
        const int h = h0 + u;
        const bool isq = h < p.H;
        const float* g = isq ? p.gq : p.gk;
        // the shuffles of the norm need the whole warp: every lane takes them when
        // either gain is given, and a vector without one keeps its values
        if (p.gq || p.gk) {
            float4 y[VPL], gv[VPL];
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int d = 4 * (gl + LPH * i);
                y[i] = x[u][i];
                gv[i] = (g && d < p.dh) ? __ldg(reinterpret_cast<const float4*>(g + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            head_norm<LPH, VPL>(y, gv, p.dh, p.eps);
            if (g)
#pragma unroll
                for (int i = 0; i < VPL; ++i) x[u][i] = y[i];
        }
        if (!live || h >= NH) continue;
        float* dst = isq ? p.qo + (size_t)row * p.ldqo + (size_t)h * p.dh
                         : p.ko + (size_t)row * p.ldko + (size_t)(h - p.H) * p.dh;
        const float sc = isq ? p.q_scale : 1.0f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int d = 4 * (gl + LPH * i);
            if (d >= p.dh) continue;
            float4 y = p.table ? rotate4(x[u][i], t[i]) : x[u][i];
            if (isq) { y.x = fmul(y.x, sc); y.y = fmul(y.y, sc); y.z = fmul(y.z, sc); y.w = fmul(y.w, sc); }
            *reinterpret_cast<float4*>(dst + d) = y;
        }
    }
}

// One lane group per (row, HPU heads). The row's table entries are loaded once for
// its HPU heads.
template <int LPH, int VPL, int HPU>
__global__ void __launch_bounds__(256) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    const int per_row = (p.H + p.KVH + HPU - 1) / HPU;
    const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) / LPH;
    const int gl = threadIdx.x % LPH;
    const long long row = unit / per_row;
    bool live = row < p.n_rows;
    int pos = 0;
    if (live && p.pos) {
        pos = __ldg(p.pos + row);
        if (pos < 0) live = false;
        else if (p.table && pos >= p.table_rows) {
            live = false;
            set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
        }
    }
    norm_rope_heads<LPH, VPL, HPU>(p, live ? (int)row : 0, (int)(unit % per_row) * HPU, gl, live, live ? pos : 0);
}

// ------------------------------------------------------------------ append
struct AppendParams {
    PagedKv c;
    PagedRows r;
    const float* k;          // [n_rows][ldk]
    const float* v;          // [n_rows][ldv]
    long long ldk, ldv;
    NormRopeParams nr;       // gains, table; its q / qo for the queries (q nullptr: none)
    int items;               // runs the grid covers
    int kv_ctas;             // grid y below this: K and V, from it on: queries
    int* err;
};

// One warp: the run's rows of one head's K or V. It holds all of them in registers
// (lane group i the rows i, i + RPW, ...), so the block's new scale is known before
// a code is written.
template <int LPH, int VPL>
__device__ __forceinline__ void append_head(const AppendParams& p, const BlockRun& run, int page, int head, bool is_k,
                                            int lane) {
    constexpr int RPW = 32 / LPH;                  // rows per pass
    constexpr int NP = kKvBlock / RPW;             // passes
    const int dh = p.c.dh, gl = lane % LPH, g = lane / LPH;
    const float* src = is_k ? p.k : p.v;
    const long long ld = is_k ? p.ldk : p.ldv;
    const bool rope = is_k && p.nr.table;
    float4 x[NP][VPL];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int i = j * RPW + g;
#pragma unroll
        for (int e = 0; e < VPL; ++e) {
            const int d = 4 * (gl + LPH * e);
            x[j][e] = (i < run.n && d < dh)
                          ? __ldg(reinterpret_cast<const float4*>(src + (size_t)(run.row + i) * ld + (size_t)head * dh + d))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    if (is_k && p.nr.gk) {
        float4 gv[VPL];
#pragma unroll
        for (int e = 0; e < VPL; ++e) {
            const int d = 4 * (gl + LPH * e);
            gv[e] = d < dh ? __ldg(reinterpret_cast<const float4*>(p.nr.gk + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j)
            if (j * RPW < run.n) head_norm<LPH, VPL>(x[j], gv, dh, p.nr.eps);
    }
    if (rope) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int i = j * RPW + g;
#pragma unroll
            for (int e = 0; e < VPL; ++e) {
                const int d = 4 * (gl + LPH * e);
                if (i < run.n && d < dh)
                    x[j][e] = rotate4(x[j][e], __ldg(reinterpret_cast<const float4*>(
                                                   p.nr.table + (size_t)(run.pos + i) * dh + d)));
            }
        }
    }
    unsigned am = 0u;                              // largest |x| as bits: a NaN or infinity is above 0x7f7fffff
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int e = 0; e < VPL; ++e)
            am = max(am, max(max(__float_as_uint(x[j][e].x) & 0x7fffffffu, __float_as_uint(x[j][e].y) & 0x7fffffffu),
                             max(__float_as_uint(x[j][e].z) & 0x7fffffffu, __float_as_uint(x[j][e].w) & 0x7fffffffu)));
    am = __reduce_max_sync(0xffffffffu, am);
    const int psz = 1 << p.c.page_log2;
    const int off = run.pos & (psz - 1), o0 = run.pos % kKvBlock;
    const size_t cell = ((size_t)page * p.c.KVH + head) * (psz / kKvBlock) + off / kKvBlock;
    float* sp = (is_k ? p.c.ks : p.c.vs) + cell;
    int8_t* codes = (is_k ? p.c.k : p.c.v) + cell * kKvBlock * dh;    // the block's 16 rows
    // a block that starts with this run has no older rows: its scale starts afresh
    const float old = o0 == 0 ? 0.0f : *sp;
    float now = am >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fdiv(__uint_as_float(am), 127.0f);
    if (!(now <= old)) {                           // grown (or NaN on either side)
        if (old != old) now = old;
        else if (now == now && o0 > 0) {           // older rows to the new scale
            const float ratio = fdiv(old, now);
            for (int b = lane * 4; b < o0 * dh; b += 128) {
                char4 w = *reinterpret_cast<char4*>(codes + b);
                w.x = (signed char)__float2int_rn(fmul((float)w.x, ratio));
                w.y = (signed char)__float2int_rn(fmul((float)w.y, ratio));
                w.z = (signed char)__float2int_rn(fmul((float)w.z, ratio));
                w.w = (signed char)__float2int_rn(fmul((float)w.w, ratio));
                *reinterpret_cast<char4*>(codes + b) = w;
            }
        }
    } else {
        now = old;
    }
    __syncwarp();
    if (lane == 0) *sp = now;
    const bool some = now > 0.0f;                  // false for a block of zeros and for a NaN scale
    auto code = [&](float v) {
        return some ? (signed char)max(-127, min(127, __float2int_rn(fdiv(v, now)))) : (signed char)0;
    };
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int i = j * RPW + g;
#pragma unroll
        for (int e = 0; e < VPL; ++e) {
            const int d = 4 * (gl + LPH * e);
            if (i < run.n && d < dh)
                *reinterpret_cast<char4*>(codes + (size_t)(o0 + i) * dh + d) =
                    make_char4(code(x[j][e].x), code(x[j][e].y), code(x[j][e].z), code(x[j][e].w));
        }
    }
}

// Grid (runs, CTAs of a run): every warp finds the run; a warp of the first kv_ctas
// takes one head's K or V of it, a group of lanes of the others 4 query vectors of a row.
template <int LPH, int VPL>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ AppendParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    BlockRun run = find_run(p.r, blockIdx.x, p.items, p.err, lane);
    if (run.s < 0) return;
    if (p.nr.table && run.pos + run.n > p.nr.table_rows) {          // rows past the table have no rotation
        if (lane == 0) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
        run.n = p.nr.table_rows - run.pos;
        if (run.n <= 0) return;
    }
    if ((int)blockIdx.y < p.kv_ctas) {
        const int task = blockIdx.y * 8 + warp;
        if (task >= 2 * p.c.KVH) return;
        const int page = page_of(p.c, p.r, run.s, run.pos);
        if (page < 0) {
            if (lane == 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
            return;
        }
        append_head<LPH, VPL>(p, run, page, task >> 1, (task & 1) == 0, lane);
        return;
    }
    constexpr int HPU = 4;
    const int per_row = (p.nr.H + HPU - 1) / HPU;
    const int unit = ((blockIdx.y - p.kv_ctas) * 256 + threadIdx.x) / LPH;
    const int i = unit / per_row;
    const bool live = i < run.n;
    norm_rope_heads<LPH, VPL, HPU>(p.nr, live ? run.row + i : 0, unit % per_row * HPU, lane % LPH, live,
                                   live ? run.pos + i : 0);
}

// ------------------------------------------------------------------ read back
struct ReadParams {
    PagedKv c;
    PagedRows r;
    void* k;                 // [n_rows][ld] f32 or bf16
    void* v;
    long long ld;
    int items;
    int* err;
};

__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Grid (runs, CTAs of 8 head tasks): a warp turns one head's K or V codes of the run
// (contiguous bytes) into values. Rows on a missing page become zeros.
template <bool BF16>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ ReadParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const BlockRun run = find_run(p.r, blockIdx.x, p.items, p.err, lane);
    if (run.s < 0) return;
    const int task = blockIdx.y * 8 + warp;
    if (task >= 2 * p.c.KVH) return;
    const int head = task >> 1, dh = p.c.dh;
    const bool is_k = (task & 1) == 0;
    const int page = page_of(p.c, p.r, run.s, run.pos);
    if (page < 0 && lane == 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
    const int psz = 1 << p.c.page_log2;
    const size_t cell = ((size_t)max(page, 0) * p.c.KVH + head) * (psz / kKvBlock) + (run.pos & (psz - 1)) / kKvBlock;
    const float s = page < 0 ? 0.0f : __ldg((is_k ? p.c.ks : p.c.vs) + cell);
    const int8_t* codes = (is_k ? p.c.k : p.c.v) + cell * kKvBlock * dh + (size_t)(run.pos % kKvBlock) * dh;
    for (int b = lane * 8; b < run.n * dh; b += 256) {
        const uint2 w = page < 0 ? make_uint2(0u, 0u) : __ldg(reinterpret_cast<const uint2*>(codes + b));
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = fmul((float)(signed char)(w.x >> (8 * e)), s);
            f[4 + e] = fmul((float)(signed char)(w.y >> (8 * e)), s);
        }
        const size_t at = (size_t)(run.row + b / dh) * p.ld + (size_t)head * dh + b % dh;
        if constexpr (BF16) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_k ? p.k : p.v) + at) =
                make_uint4(bf16x2_bits(f[0], f[1]), bf16x2_bits(f[2], f[3]), bf16x2_bits(f[4], f[5]), bf16x2_bits(f[6], f[7]));
        } else {
            float* o = static_cast<float*>(is_k ? p.k : p.v) + at;
            *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
}

// ------------------------------------------------------------------ attention
// The codes are exact small integers, so both products run as integer dots on the
// tensor cores (warp-level s8 MMAs) with the f32 side split into three signed
// base-256 digits: X = rint(x 2^..) with |X| <= kDigitMax = d2 65536 + d1 256 + d0,
// 23 bits below the row's largest element. The digit sums are exact in int32 and
// are joined in f32, so a score or an output carries the error of one 23-bit
// rounding per factor instead of a chain of f32 roundings, at a third of the int8
// rate and without converting a single code.
// three digits in [-128, 127] reach 2^23 - 1 - 0x8080 = 8355711; a little below it,
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

// two f32 in one instruction: the attention kernels are bound by what the schedulers
// issue, and a packed operation takes one slot for two (same rounding)
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
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

// d2 65536 + d1 256 + d0 of two neighbouring sums (elements y, y + 1 of the fragments):
// the lower two joined as integers (256 products: below 2^30)
__device__ __forceinline__ f32x2 join_digits(const int (&c)[3][4], int y) {
    return fma2(pack2((float)c[2][y], (float)c[2][y + 1]), pack2(65536.0f, 65536.0f),
                pack2((float)(c[1][y] * 256 + c[0][y]), (float)(c[1][y + 1] * 256 + c[0][y + 1])));
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the factor that takes values up to `top` (>= 0) to integers up to kDigitMax; tiny
// tops (below 1e-31) keep fewer bits, 0 gives 0, NaN and infinity NaN
__device__ __forceinline__ float digit_factor(float top) {
    if (!(top < __int_as_float(0x7f800000))) return __int_as_float(0x7fffffff);
    return top > 0.0f ? fminf(fdiv((float)kDigitMax, top), 0x1p126f) : 0.0f;
}

struct PagedAttnParams {
    PagedKv c;
    PagedRows r;
    const float* q;          // [n_rows][ldq], rotated and pre-scaled
    float* out;              // [n_rows][ldo]
    long long ldq, ldo;
    int H, G;                // G = H / KVH
    int kc;                  // keys per split
    int nsplit;              // splits of a sequence of cap keys
    float* part;             // [n_rows][H][nsplit][dh + 4]: o, m (base 2), l
    int* err;
};

// A unit of attention work: columns col0 .. of one KV head's (row, head) pairs of a
// sequence, against keys of split `split`.
struct AttnItem {
    int s, a, len, kv;       // sequence and its rows (s < 0: none left)
    int kvh, tile, split;
};

__device__ __forceinline__ long long shfl64(unsigned m, long long v, int src) {
    return (long long)(((unsigned long long)(unsigned)__shfl_sync(m, (int)(v >> 32), src) << 32) |
                       (unsigned)__shfl_sync(m, (int)v, src));
}

// splits of n keys (at least one: it also writes rows that see none)
__device__ __forceinline__ int splits_of(const PagedAttnParams& p, int n) { return max((n + p.kc - 1) / p.kc, 1); }

// item number `item` of the call (tiles of NC columns), found by one warp
template <int NC>
__device__ __forceinline__ AttnItem find_item(const PagedAttnParams& p, long long item, int lane) {
    AttnItem out{-1, 0, 0, 0, 0, 0, 0};
    long long before = 0;
    for (int base = 0; base < p.r.n_seq; base += 32) {
        const int s = base + lane;
        SeqRows q{0, 0, 0};
        long long cnt = 0;
        int tiles = 0;
        if (s < p.r.n_seq) {
            q = seq_rows(p.r, s);
            if (q.len > 0) {
                if (q.kv > p.r.cap) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
                const int n = min(q.kv, p.r.cap);
                tiles = (q.len * p.G + NC - 1) / NC;
                cnt = (long long)tiles * p.c.KVH * splits_of(p, n);
            }
        }
        long long incl = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = shfl64(0xffffffffu, incl, (lane - o) & 31);
            if (lane >= o) incl += v;
        }
        const long long total = shfl64(0xffffffffu, incl, 31);
        if (item < before + total) {
            const int src = __ffs(__ballot_sync(0xffffffffu, before + incl > item)) - 1;
            const long long idx = item - before - shfl64(0xffffffffu, incl - cnt, src);
            out.s = base + src;
            out.a = __shfl_sync(0xffffffffu, q.a, src);
            out.len = __shfl_sync(0xffffffffu, q.len, src);
            out.kv = __shfl_sync(0xffffffffu, q.kv, src);
            // the last rows first: with causal lengths they are the longest
            const int splits = splits_of(p, min(out.kv, p.r.cap));
            const long long rest = idx / p.c.KVH;
            out.kvh = (int)(idx % p.c.KVH);
            out.split = (int)(rest % splits);
            out.tile = __shfl_sync(0xffffffffu, tiles, src) - 1 - (int)(rest / splits);
            return out;
        }
        before += total;
    }
    return out;
}

// splits that a row at position pos has
__device__ __forceinline__ int row_splits(const PagedAttnParams& p, int pos) {
    return splits_of(p, min(pos + 1, p.r.cap));
}

// One query row (16 lanes, lane l16 the elements 4 l16 + 64 i ..) as digits: store(e, d,
// word) takes digit e of elements d .. d + 3. *unit = the score of one integer unit in
// base 2, NaN for a row that is not finite, 0 for one of zeros (`live` false: zeros).
template <int DP, typename Store>
__device__ __forceinline__ void query_digits(const float* qr, bool live, int dh, int l16, Store store, float* unit) {
    constexpr int NE = DP / 64;
    float4 x[NE];
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int d = 4 * (l16 + 16 * i);
        x[i] = (live && d < dh) ? __ldg(reinterpret_cast<const float4*>(qr + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        bad |= x[i].x != x[i].x || x[i].y != x[i].y || x[i].z != x[i].z || x[i].w != x[i].w;
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = digit_factor(top);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        uint32_t w[3];
        digits4(digit_bits(x[i].x, f), digit_bits(x[i].y, f), digit_bits(x[i].z, f), digit_bits(x[i].w, f), w);
#pragma unroll
        for (int e = 0; e < 3; ++e) store(e, 4 * (l16 + 16 * i), w[e]);
    }
    if (l16 == 0) *unit = f > 0.0f ? __fdividef(1.4426950408889634f, f) : f;   // log2 e
}

// ---- few rows per sequence: a CTA of 4 warps takes 8 columns (token, head) of one KV
// head against one split of the keys; warp w the 32-key steps w, w + 4, .... The codes
// go from global memory straight into MMA fragments (A = keys x d for the scores,
// d x keys for the output), so a warp keeps 64 * dh bytes of loads in flight and
// nothing is staged; the four warps' (m, l, o) meet in shared memory.
constexpr int kSplitWarps = 4;
constexpr int kSplitCols = 8;

template <int DP>
struct SplitShape {
    static constexpr int NH = DP / 64;             // 64-byte parts of a key row
    static constexpr int VW = DP / 32;             // 32-bit words of a value row that a lane holds
    static constexpr int NM = DP / 16;             // output tiles of 16 elements
    static constexpr int QBytes = 3 * kSplitCols * DP;
    static constexpr int WStride = 36;             // ints; column rows 4 banks apart
    static constexpr int MergeFloats = kSplitWarps * kSplitCols * (DP + 2);
    static constexpr int WBytes = kSplitWarps * kSplitCols * WStride * 4;
    static constexpr int Smem = QBytes + WBytes + MergeFloats * 4 + 64;
};

template <int DP>
__global__ void __launch_bounds__(kSplitWarps * 32, DP == 256 ? 2 : 4)
paged_attn_split_kernel(const __grid_constant__ PagedAttnParams p) {
    using Sh = SplitShape<DP>;
    extern __shared__ __align__(16) unsigned char ps_raw[];
    uint8_t* qd = ps_raw;                                                  // [3][8][DP] digits of the queries
    float* sq = reinterpret_cast<float*>(ps_raw + Sh::QBytes);             // [8] their units (log2 e in)
    uint32_t* wx = reinterpret_cast<uint32_t*>(ps_raw + Sh::QBytes + 64);            // [4][8][WStride] weights
    float* mo = reinterpret_cast<float*>(ps_raw + Sh::QBytes + 64 + Sh::WBytes);   // [4][8][DP]
    float* ml = mo + kSplitWarps * kSplitCols * DP;                        // [4][8][2]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int dh = p.c.dh, psz = 1 << p.c.page_log2;
    uint32_t* wxw = wx + warp * kSplitCols * Sh::WStride;

    for (long long item = blockIdx.x;; item += gridDim.x) {
        const AttnItem it = find_item<kSplitCols>(p, item, lane);
        if (it.s < 0) return;
        const int cols = min(it.len * p.G - it.tile * kSplitCols, kSplitCols);
        const int col0 = it.tile * kSplitCols;                             // column = token * G + head
        const int pos_last = it.kv - it.len + (col0 + cols - 1) / p.G;     // of the tile's last row
        const int n = min(pos_last + 1, p.r.cap);                          // keys that any column sees
        const int j0 = it.split * p.kc;
        if (j0 >= n && it.split > 0) continue;                             // the tile ends before this split
        const int jend = min(n, j0 + p.kc);

        // queries -> digits: 16 lanes a column
        {
            const int col = tid >> 4, cc = col0 + col;
            query_digits<DP>(p.q + (size_t)(it.a + cc / p.G) * p.ldq + (size_t)(it.kvh * p.G + cc % p.G) * dh, col < cols, dh,
                             tid & 15, [&](int e, int d, uint32_t w) {
                                 *reinterpret_cast<uint32_t*>(qd + (e * kSplitCols + col) * DP + d) = w;
                             }, sq + col);
        }
        __syncthreads();
        uint32_t qb[3][Sh::NH][4];                                         // B fragments of column g
#pragma unroll
        for (int e = 0; e < 3; ++e)
#pragma unroll
            for (int h = 0; h < Sh::NH; ++h) {
                const uint4 w = lds128(qd + (e * kSplitCols + g) * DP + 64 * h + 16 * t);
                qb[e][h][0] = w.x; qb[e][h][1] = w.y; qb[e][h][2] = w.z; qb[e][h][3] = w.w;
            }
        const float sq0 = sq[2 * t], sq1 = sq[2 * t + 1];
        // keys that columns 2t and 2t + 1 see
        const int pos0 = it.kv - it.len;
        const int lim0 = 2 * t < cols ? min(pos0 + (col0 + 2 * t) / p.G + 1, n) : 0;
        const int lim1 = 2 * t + 1 < cols ? min(pos0 + (col0 + 2 * t + 1) / p.G + 1, n) : 0;

        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;        // running max; this lane's part of the sum
        f32x2 o[Sh::NM][2];                                                // elements, columns (2t, 2t + 1)
#pragma unroll
        for (int i = 0; i < Sh::NM; ++i) o[i][0] = o[i][1] = 0ull;

        for (int j = j0 + warp * 32; j < jend; j += kSplitWarps * 32) {
            // the step's two blocks: where they are and their scales
            size_t at[2];
            float sk[2], sv[2];
            bool there[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int jb = j + 16 * b;
                const int page = jb < jend ? page_of(p.c, p.r, it.s, jb) : -1;
                there[b] = page >= 0;
                if (jb < jend && page < 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
                const size_t cell = ((size_t)max(page, 0) * p.c.KVH + it.kvh) * (psz >> 4) + ((jb & (psz - 1)) >> 4);
                at[b] = cell * kKvBlock * dh;
                sk[b] = there[b] ? __ldg(p.c.ks + cell) : 0.0f;
                sv[b] = there[b] ? __ldg(p.c.vs + cell) : 0.0f;
            }
            uint4 kf[2][2][Sh::NH];                                        // [block][row g, g + 8][part]
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int h = 0; h < Sh::NH; ++h) {
                        const int d = 64 * h + 16 * t;
                        kf[b][r][h] = (there[b] && d < dh)
                                          ? __ldg(reinterpret_cast<const uint4*>(p.c.k + at[b] + (size_t)(g + 8 * r) * dh + d))
                                          : make_uint4(0u, 0u, 0u, 0u);
                    }
            uint32_t vf[2][4][Sh::VW];                                     // [block][key 4t + i][words]
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int8_t* vr = p.c.v + at[b] + (size_t)(4 * t + i) * dh;
                    if constexpr (Sh::VW == 2) {
                        const int d = 8 * g;
                        const uint2 w = (there[b] && d < dh) ? __ldg(reinterpret_cast<const uint2*>(vr + d)) : make_uint2(0u, 0u);
                        vf[b][i][0] = w.x; vf[b][i][1] = w.y;
                    } else {
#pragma unroll
                        for (int u = 0; u < Sh::VW / 4; ++u) {
                            const int d = (DP / 8) * g + 16 * u;
                            const uint4 w = (there[b] && d < dh) ? __ldg(reinterpret_cast<const uint4*>(vr + d))
                                                                 : make_uint4(0u, 0u, 0u, 0u);
                            vf[b][i][4 * u] = w.x; vf[b][i][4 * u + 1] = w.y; vf[b][i][4 * u + 2] = w.z; vf[b][i][4 * u + 3] = w.w;
                        }
                    }
                }

            // scores (base 2): rows g, g + 8 of each block, columns 2t, 2t + 1
            float s[2][4];
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                int c[3][4];
#pragma unroll
                for (int h = 0; h < Sh::NH; ++h)
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        if (h == 0) mma_s8_first(c[e], kf[b][0][h].x, kf[b][1][h].x, kf[b][0][h].y, kf[b][1][h].y, qb[e][h][0], qb[e][h][1]);
                        else mma_s8(c[e], kf[b][0][h].x, kf[b][1][h].x, kf[b][0][h].y, kf[b][1][h].y, qb[e][h][0], qb[e][h][1]);
                        mma_s8(c[e], kf[b][0][h].z, kf[b][1][h].z, kf[b][0][h].w, kf[b][1][h].w, qb[e][h][2], qb[e][h][3]);
                    }
                const f32x2 u = pack2(sq0 * sk[b], sq1 * sk[b]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int key = j + 16 * b + 8 * r + g;
                    const float2 a = unpack2(mul2(join_digits(c, 2 * r), u));
                    s[b][2 * r] = there[b] && key < lim0 ? a.x : -INFINITY;
                    s[b][2 * r + 1] = there[b] && key < lim1 ? a.y : -INFINITY;
                    mx0 = fmaxf(mx0, s[b][2 * r]);
                    mx1 = fmaxf(mx1, s[b][2 * r + 1]);
                }
            }
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
            }
            const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
            const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
            const float back0 = exp2_fast(m0 - b0), back1 = exp2_fast(m1 - b1);
            m0 = n0; m1 = n1;
            l0 *= back0; l1 *= back1;
            // weights p v_scale; -inf scores (masked) give 0 even where a scale is NaN
            float wt0 = 0.0f, wt1 = 0.0f;                                  // largest weights; NaN if one is
            bool nan0 = false, nan1 = false;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float e0 = exp2_fast(s[b][2 * r] - b0), e1 = exp2_fast(s[b][2 * r + 1] - b1);
                    l0 += e0; l1 += e1;
                    const float w0 = s[b][2 * r] == -INFINITY ? 0.0f : e0 * sv[b];
                    const float w1 = s[b][2 * r + 1] == -INFINITY ? 0.0f : e1 * sv[b];
                    s[b][2 * r] = w0; s[b][2 * r + 1] = w1;
                    wt0 = fmaxf(wt0, w0); wt1 = fmaxf(wt1, w1);
                    nan0 |= w0 != w0; nan1 |= w1 != w1;
                }
            if (nan0) wt0 = INFINITY;
            if (nan1) wt1 = INFINITY;
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
                wt0 = fmaxf(wt0, __shfl_xor_sync(0xffffffffu, wt0, x));
                wt1 = fmaxf(wt1, __shfl_xor_sync(0xffffffffu, wt1, x));
            }
            const float f0 = digit_factor(wt0), f1 = digit_factor(wt1);
            __syncwarp();
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    wxw[2 * t * Sh::WStride + 16 * b + 8 * r + g] = digit_bits_pos(s[b][2 * r], f0);
                    wxw[(2 * t + 1) * Sh::WStride + 16 * b + 8 * r + g] = digit_bits_pos(s[b][2 * r + 1], f1);
                }
            __syncwarp();
            uint32_t wb[2][3];                                             // B fragments: keys 4t .., 16 + 4t .. of column g
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint4 w = lds128(wxw + g * Sh::WStride + 16 * b + 4 * t);
                digits4(w.x, w.y, w.z, w.w, wb[b]);
            }
            const f32x2 u = pack2(f0 > 0.0f ? __fdividef(1.0f, f0) : f0, f1 > 0.0f ? __fdividef(1.0f, f1) : f1);
            const f32x2 back = pack2(back0, back1);
            // output elements (DP / 8) g + 2 m, + 1 (rows g and g + 8 of tile m): four keys' bytes of one element
            // make one A register
#pragma unroll
            for (int w = 0; w < Sh::VW; ++w) {
                uint32_t a[2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint32_t x = __byte_perm(vf[b][0][w], vf[b][1][w], 0x5140), y = __byte_perm(vf[b][2][w], vf[b][3][w], 0x5140);
                    const uint32_t z = __byte_perm(vf[b][0][w], vf[b][1][w], 0x7362), v = __byte_perm(vf[b][2][w], vf[b][3][w], 0x7362);
                    a[b][0] = __byte_perm(x, y, 0x5410); a[b][1] = __byte_perm(x, y, 0x7632);
                    a[b][2] = __byte_perm(z, v, 0x5410); a[b][3] = __byte_perm(z, v, 0x7632);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    int c[3][4];
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        mma_s8_first(c[e], a[0][2 * k], a[0][2 * k + 1], a[1][2 * k], a[1][2 * k + 1], wb[0][e], wb[1][e]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[2 * w + k][i] = fma2(join_digits(c, 2 * i), u, mul2(o[2 * w + k][i], back));
                }
            }
        }
        // this warp's columns: sum over the lanes of a column, then all to shared memory
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            l1 += __shfl_xor_sync(0xffffffffu, l1, x);
        }
        if (g == 0) {
            float* q = ml + (warp * kSplitCols + 2 * t) * 2;
            q[0] = m0; q[1] = l0; q[2] = m1; q[3] = l1;
        }
        float* ow = mo + warp * kSplitCols * DP;
#pragma unroll
        for (int i = 0; i < Sh::NM; ++i) {
            const int d = (DP / 8) * g + 2 * i;
            const float2 x = unpack2(o[i][0]), y = unpack2(o[i][1]);
            *reinterpret_cast<float2*>(ow + (2 * t) * DP + d) = make_float2(x.x, y.x);
            *reinterpret_cast<float2*>(ow + (2 * t + 1) * DP + d) = make_float2(x.y, y.y);
        }
        __syncthreads();
        for (int i = tid; i < cols * (DP / 4); i += kSplitWarps * 32) {
            const int col = i / (DP / 4), d = 4 * (i % (DP / 4)), cc = col0 + col;
            const int pos = pos0 + cc / p.G, splits = row_splits(p, pos);
            if (d >= dh || it.split >= splits) continue;
            float M = -INFINITY, L = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kSplitWarps; ++w) M = fmaxf(M, ml[(w * kSplitCols + col) * 2]);
            const float B = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < kSplitWarps; ++w) {
                const float e = exp2_fast(ml[(w * kSplitCols + col) * 2] - B);
                const float4 x = lds128f(mo + (w * kSplitCols + col) * DP + d);
                L = ffma(ml[(w * kSplitCols + col) * 2 + 1], e, L);
                acc.x = ffma(x.x, e, acc.x); acc.y = ffma(x.y, e, acc.y);
                acc.z = ffma(x.z, e, acc.z); acc.w = ffma(x.w, e, acc.w);
            }
            const int row = it.a + cc / p.G, h = it.kvh * p.G + cc % p.G;
            if (splits == 1) {
                const float inv = L == 0.0f ? 0.0f : fdiv(1.0f, L);
                *reinterpret_cast<float4*>(p.out + (size_t)row * p.ldo + (size_t)h * dh + d) =
                    make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                float* pp = p.part + (((size_t)row * p.H + h) * p.nsplit + it.split) * (dh + 4);
                *reinterpret_cast<float4*>(pp + d) = acc;
                if (d == 0) { pp[dh] = M; pp[dh + 1] = L; }
            }
        }
        __syncthreads();
    }
}

// ---- many rows per sequence: a CTA of 4 warps takes 64 rows ((token, head) pairs of
// one KV head), warp w 16 of them, against a split of the keys in tiles of KT. A =
// query or weight digits (rows x 32), B = codes: keys as they lie, values turned to
// [d][key] on their way into shared memory (byte permutes, once for the CTA). The
// key order inside a B fragment of the values is the one that the score fragments
// already have, so weights go from scores to A fragments inside their thread.
// Codes of tile i + 1 are on their way while tile i is computed. Every tile ends with
// folding the output's digit sums into f32 (their unit changes with the row's
// maximum), which is why KT is as large as the registers allow.
constexpr int kTileRows = 64;

template <int DP>
struct TileShape {
    static constexpr int KT = DP == 256 ? 64 : 128;            // keys per tile
    static constexpr int NB = KT / 16;                         // blocks per tile
    static constexpr int NH = DP / 64;
    static constexpr int NT = DP / 8;                          // output tiles of 8 elements
    static constexpr int QBytes = 3 * kTileRows * DP;
    static constexpr int KBytes = KT * DP;
    static constexpr int Smem = QBytes + 4 * KBytes + kTileRows * 4 + 2 * 3 * NB * 4 + 2 * NB * 8;
};

// byte offset of 16-byte unit u of row `row` of `width` bytes: swapped between halves in
// odd rows so that the fragment loads of two neighbouring rows meet no bank twice
template <int width>
__device__ __forceinline__ int unit_at(int row, int u) {
    return row * width + 16 * (width >= 128 ? u ^ ((row & 1) << 2) : u);
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int DP>
__global__ void __launch_bounds__(128, DP == 256 ? 1 : 2) paged_attn_tile_kernel(const __grid_constant__ PagedAttnParams p) {
    using Sh = TileShape<DP>;
    constexpr int KT = Sh::KT, NB = Sh::NB;
    extern __shared__ __align__(16) unsigned char pt_raw[];
    uint8_t* qd = pt_raw;                                      // A fragments [3][4 warps][DP / 32][lane][16]
    uint8_t* kt = qd + Sh::QBytes;                             // [2][KT][DP]
    uint8_t* vt = kt + 2 * Sh::KBytes;                         // [2][DP][KT]
    float* sq = reinterpret_cast<float*>(vt + 2 * Sh::KBytes); // [64]
    float* sc = sq + kTileRows;                                // [2][3][NB]: key scales, value scales, 1 where there
    long long* cell = reinterpret_cast<long long*>(sc + 6 * NB);   // [2][NB] a tile's blocks in the pool
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int dh = p.c.dh, psz = 1 << p.c.page_log2;

    const AttnItem it = find_item<kTileRows>(p, blockIdx.x, lane);
    if (it.s < 0) return;
    const int row0 = it.tile * kTileRows, rows = min(it.len * p.G - row0, kTileRows);
    const int pos0 = it.kv - it.len;
    const int n = min(pos0 + (row0 + rows - 1) / p.G + 1, p.r.cap);      // keys that any row sees
    const int j0 = it.split * p.kc, jend = min(n, j0 + p.kc);
    if (j0 >= n && it.split > 0) return;
    const int ntiles = max((jend - j0 + KT - 1) / KT, 0);

    // a block's number in the pool (its codes start at 16 dh times that); -1: page outside
    // the pool, -2: past the end
    auto cell_at = [&](int j) -> long long {
        if (j >= jend) return -2;
        const int page = page_of(p.c, p.r, it.s, j);
        return page < 0 ? -1 : ((long long)page * p.c.KVH + it.kvh) * (psz >> 4) + ((j & (psz - 1)) >> 4);
    };
    if (tid < 2 * NB && ntiles > 0) cell[tid] = cell_at(j0 + 16 * tid);

    // queries -> digits: 16 lanes a row
#pragma unroll 1
    for (int r = tid >> 4; r < kTileRows; r += 8) {
        const int l16 = tid & 15, cc = row0 + r;
        const float* qr = p.q + (size_t)(it.a + cc / p.G) * p.ldq + (size_t)(it.kvh * p.G + cc % p.G) * dh;
        query_digits<DP>(qr, r < rows, dh, l16, [&](int e, int d, uint32_t w) {
            // elements d .. d + 3: lane 4 (row & 7) + quad of the row's 16-byte unit, word by row half and k half
            const int step = 2 * (d >> 6) + ((d >> 3) & 1), word = ((r >> 3) & 1) + 2 * ((d >> 2) & 1);
            *reinterpret_cast<uint32_t*>(qd + (((e * 4 + (r >> 4)) * (DP / 32) + step) * 32 + 4 * (r & 7) + ((d >> 4) & 3)) * 16 + 4 * word) = w;
        }, sq + r);
    }
    __syncthreads();

    auto load_keys = [&](int i) {                              // and the scales
        const int b = i & 1;
        uint8_t* kd = kt + b * Sh::KBytes;
#pragma unroll
        for (int x = 0; x < KT * DP / 16 / 128; ++x) {
            const int unit = x * 128 + tid, key = unit / (DP / 16), u = unit % (DP / 16);
            const long long at = cell[NB * b + (key >> 4)];
            const bool there = at >= 0 && 16 * u < dh;
            cp_async16(kd + unit_at<DP>(key, u), p.c.k + (there ? at * (kKvBlock * dh) + (key & 15) * dh + 16 * u : 0), there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (tid < 2 * NB) {
            const long long cb = cell[NB * b + tid % NB];
            sc[3 * NB * b + tid] = cb >= 0 ? __ldg((tid < NB ? p.c.ks : p.c.vs) + cb) : 0.0f;
            if (tid < NB) sc[3 * NB * b + 2 * NB + tid] = cb >= 0 ? 1.0f : 0.0f;
            if (cb == -1) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
        }
    };
    // This thread's part of a value tile: in block vb four keys vq2 + {0, 1, 8, 9} of 16
    // elements from d0 + 16 x. The lanes of a warp cover 32 (block, key group) pairs of one
    // 16-element column (KT = 128), so that its word stores meet no bank twice.
    constexpr int VH = KT / 64;                                // 64-key halves among a warp's lanes
    constexpr int VC = KT * DP / 64 / 128;                     // 16-byte columns a thread turns
    const int vb = (lane & 15) >> 2, vq2 = (lane & 3) * 2, vh = VH == 2 ? lane >> 4 : 0;
    const int d0 = 16 * (VH == 2 ? VC * warp : VC * (2 * warp + (lane >> 4)));
    uint4 vr[VC][4];
    auto load_values = [&](int i) {
        const long long at = cell[NB * (i & 1) + 4 * vh + vb];
#pragma unroll
        for (int x = 0; x < VC; ++x) {
            const int d = d0 + 16 * x;
            const bool there = at >= 0 && d < dh;
            const int8_t* src = p.c.v + (there ? at * (kKvBlock * dh) + vq2 * dh + d : 0);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                vr[x][k] = there ? __ldg(reinterpret_cast<const uint4*>(src + ((k >> 1) * 8 + (k & 1)) * dh)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto store_values = [&](int i) {
        uint8_t* vd = vt + (i & 1) * Sh::KBytes;
#pragma unroll
        for (int x = 0; x < VC; ++x) {
            const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vr[x][0]);
            const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vr[x][1]);
            const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vr[x][2]);
            const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vr[x][3]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t a = __byte_perm(w0[w], w1[w], 0x5140), b = __byte_perm(w2[w], w3[w], 0x5140);
                const uint32_t c = __byte_perm(w0[w], w1[w], 0x7362), e = __byte_perm(w2[w], w3[w], 0x7362);
                const uint32_t y[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, e, 0x5410),
                                       __byte_perm(c, e, 0x7632)};
#pragma unroll
                for (int z = 0; z < 4; ++z)
                    *reinterpret_cast<uint32_t*>(vd + unit_at<KT>(d0 + 16 * x + 4 * w + z, 4 * vh + (vq2 >> 1)) + 4 * vb) = y[z];
            }
        }
    };

    // rows ra = 16 warp + g and ra + 8
    const int ra = 16 * warp + g;
    const int lim0 = ra < rows ? min(pos0 + (row0 + ra) / p.G + 1, n) : 0;
    const int lim1 = ra + 8 < rows ? min(pos0 + (row0 + ra + 8) / p.G + 1, n) : 0;
    int wmin = min(lim0, lim1), wmax = max(lim0, lim1);        // of the warp's rows
    wmin = __reduce_min_sync(0xffffffffu, wmin);
    wmax = __reduce_max_sync(0xffffffffu, wmax);
    const float sq0 = sq[ra], sq1 = sq[ra + 8];
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    f32x2 o[Sh::NT][2];                                        // elements 8 x + 2t, + 1 of rows ra, ra + 8
#pragma unroll
    for (int i = 0; i < Sh::NT; ++i) o[i][0] = o[i][1] = 0ull;

    if (ntiles > 0) {
        load_keys(0);
        load_values(0);
        store_values(0);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
    }
#pragma unroll 1
    for (int i = 0; i < ntiles; ++i) {
        const int j = j0 + i * KT;
        const bool more = i + 1 < ntiles;
        if (more) load_keys(i + 1);
        const bool busy = wmax > j;                            // the warp has a row that sees the tile
        uint32_t wa[KT / 32][3][4];                            // weight digits: A fragments [32 keys][digit]
        float back0 = 1.0f, back1 = 1.0f, u0 = 0.0f, u1 = 0.0f;
        if (busy) {
            const uint8_t* kd = kt + (i & 1) * Sh::KBytes;
            const float* scb = sc + 3 * NB * (i & 1);
            float2 s[KT / 8][2];                               // keys 8 x + 2t, + 1 of rows ra, ra + 8
#pragma unroll
            for (int part = 0; part < KT / 32; ++part) {       // 32 keys at a time
                int c[4][3][4];
#pragma unroll
                for (int h = 0; h < Sh::NH; ++h) {
                    uint4 b[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        b[x] = *reinterpret_cast<const uint4*>(kd + unit_at<DP>(32 * part + 8 * x + g, 4 * h + t));
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        const uint8_t* qa = qd + (((e * 4 + warp) * (DP / 32) + 2 * h) * 32 + lane) * 16;
                        const uint4 a0 = *reinterpret_cast<const uint4*>(qa), a1 = *reinterpret_cast<const uint4*>(qa + 512);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (h == 0) mma_s8_first(c[x][e], a0.x, a0.y, a0.z, a0.w, b[x].x, b[x].y);
                            else mma_s8(c[x][e], a0.x, a0.y, a0.z, a0.w, b[x].x, b[x].y);
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) mma_s8(c[x][e], a1.x, a1.y, a1.z, a1.w, b[x].z, b[x].w);
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float u = scb[2 * part + (x >> 1)];
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        s[4 * part + x][r] = unpack2(mul2(join_digits(c[x], 2 * r), pack2((r ? sq1 : sq0) * u, (r ? sq1 : sq0) * u)));
                }
            }
            float there = 0.0f, svs = 0.0f;
#pragma unroll
            for (int x = 0; x < NB; ++x) { svs += scb[NB + x]; there += scb[2 * NB + x]; }
            if (j + KT > wmin || there != (float)NB) {
#pragma unroll
                for (int x = 0; x < KT / 8; ++x)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int key = j + 8 * x + 2 * t, lim = scb[2 * NB + (x >> 1)] != 0.0f ? (r ? lim1 : lim0) : 0;
                        if (key >= lim) s[x][r].x = -INFINITY;
                        if (key + 1 >= lim) s[x][r].y = -INFINITY;
                    }
            }
            float mx0 = m0, mx1 = m1;
#pragma unroll
            for (int x = 0; x < KT / 8; ++x) {
                mx0 = fmaxf(mx0, fmaxf(s[x][0].x, s[x][0].y));
                mx1 = fmaxf(mx1, fmaxf(s[x][1].x, s[x][1].y));
            }
#pragma unroll
            for (int x = 1; x <= 2; x <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
            }
            const float b0 = mx0 == -INFINITY ? 0.0f : mx0, b1 = mx1 == -INFINITY ? 0.0f : mx1;
            back0 = exp2_fast(m0 - b0); back1 = exp2_fast(m1 - b1);
            m0 = mx0; m1 = mx1;
            // weights p v_scale. A score that is not a number makes l NaN, which is enough; a
            // value scale that is not one needs checks
            f32x2 ls0 = 0ull, ls1 = 0ull;
#pragma unroll
            for (int x = 0; x < KT / 8; ++x)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float2 z = unpack2(add2(pack2(s[x][r].x, s[x][r].y), pack2(r ? -b1 : -b0, r ? -b1 : -b0)));
                    const f32x2 ev = pack2(exp2_fast(z.x), exp2_fast(z.y));
                    if (r) ls1 = add2(ls1, ev); else ls0 = add2(ls0, ev);
                    s[x][r] = unpack2(ev);
                }
            l0 = ffma(l0, back0, unpack2(ls0).x + unpack2(ls0).y);
            l1 = ffma(l1, back1, unpack2(ls1).x + unpack2(ls1).y);
            float wt0 = 0.0f, wt1 = 0.0f;
            if (svs == svs) {
#pragma unroll
                for (int x = 0; x < KT / 8; ++x)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        s[x][r] = unpack2(mul2(pack2(s[x][r].x, s[x][r].y), pack2(scb[NB + (x >> 1)], scb[NB + (x >> 1)])));
                        if (r) wt1 = fmaxf(wt1, fmaxf(s[x][r].x, s[x][r].y)); else wt0 = fmaxf(wt0, fmaxf(s[x][r].x, s[x][r].y));
                    }
            } else {
#pragma unroll
                for (int x = 0; x < KT / 8; ++x)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // a key that is masked weighs nothing, whatever its scale
                        const int key = j + 8 * x + 2 * t, lim = r ? lim1 : lim0;
                        s[x][r].x = key < lim ? s[x][r].x * scb[NB + (x >> 1)] : 0.0f;
                        s[x][r].y = key + 1 < lim ? s[x][r].y * scb[NB + (x >> 1)] : 0.0f;
                        float& wt = r ? wt1 : wt0;
                        wt = s[x][r].x != s[x][r].x || s[x][r].y != s[x][r].y ? INFINITY : fmaxf(wt, fmaxf(s[x][r].x, s[x][r].y));
                    }
            }
#pragma unroll
            for (int x = 1; x <= 2; x <<= 1) {
                wt0 = fmaxf(wt0, __shfl_xor_sync(0xffffffffu, wt0, x));
                wt1 = fmaxf(wt1, __shfl_xor_sync(0xffffffffu, wt1, x));
            }
            const float f0 = digit_factor(wt0), f1 = digit_factor(wt1);
            u0 = f0 > 0.0f ? __fdividef(1.0f, f0) : f0;
            u1 = f1 > 0.0f ? __fdividef(1.0f, f1) : f1;
#pragma unroll
            for (int ks = 0; ks < KT / 32; ++ks)
#pragma unroll
                for (int b = 0; b < 2; ++b)                    // 16 keys: registers 2 b (row ra) and 2 b + 1 (row ra + 8)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const f32x2 f = pack2(r ? f1 : f0, r ? f1 : f0), base = pack2(kDigitBase, kDigitBase);
                        const float2 x0 = s[4 * ks + 2 * b][r], x1 = s[4 * ks + 2 * b + 1][r];
                        const float2 y0 = unpack2(fma2(pack2(x0.x, x0.y), f, base)), y1 = unpack2(fma2(pack2(x1.x, x1.y), f, base));
                        uint32_t dg[3];
                        digits4(__float_as_uint(y0.x), __float_as_uint(y0.y), __float_as_uint(y1.x), __float_as_uint(y1.y), dg);
#pragma unroll
                        for (int e = 0; e < 3; ++e) wa[ks][e][2 * b + r] = dg[e];
                    }
        }
        if (more) load_values(i + 1);                          // into registers while the output is computed
        if (busy) {
            const uint8_t* vd = vt + (i & 1) * Sh::KBytes;
#pragma unroll
            for (int x = 0; x < Sh::NT; x += 2) {              // two output tiles at a time: six independent chains
                int c[2][3][4];
#pragma unroll
                for (int h = 0; h < VH; ++h) {
                    uint4 b[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) b[z] = *reinterpret_cast<const uint4*>(vd + unit_at<KT>(8 * (x + z) + g, 4 * h + t));
#pragma unroll
                    for (int e = 0; e < 3; ++e)
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint32_t(&a)[4] = wa[2 * h][e];
                            if (h == 0) mma_s8_first(c[z][e], a[0], a[1], a[2], a[3], b[z].x, b[z].y);
                            else mma_s8(c[z][e], a[0], a[1], a[2], a[3], b[z].x, b[z].y);
                        }
#pragma unroll
                    for (int e = 0; e < 3; ++e)
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint32_t(&a)[4] = wa[2 * h + 1][e];
                            mma_s8(c[z][e], a[0], a[1], a[2], a[3], b[z].z, b[z].w);
                        }
                }
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        o[x + z][r] = fma2(join_digits(c[z], 2 * r), pack2(r ? u1 : u0, r ? u1 : u0),
                                           mul2(o[x + z][r], pack2(r ? back1 : back0, r ? back1 : back0)));
            }
        }
        if (more) {
            store_values(i + 1);
            // blocks of tile i + 2 (those of tile i are not needed any more)
            if (tid < NB) cell[NB * (i & 1) + tid] = cell_at(j + 2 * KT + 16 * tid);
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, x);
        l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int rr = ra + 8 * r, cc = row0 + rr;
        if (rr >= rows) continue;
        const int splits = row_splits(p, pos0 + cc / p.G);
        if (it.split >= splits) continue;
        const int row = it.a + cc / p.G, h = it.kvh * p.G + cc % p.G;
        const float L = r ? l1 : l0, inv = splits > 1 ? 1.0f : L == 0.0f ? 0.0f : fdiv(1.0f, L);
        float* dst = splits > 1 ? p.part + (((size_t)row * p.H + h) * p.nsplit + it.split) * (dh + 4)
                                : p.out + (size_t)row * p.ldo + (size_t)h * dh;
#pragma unroll
        for (int x = 0; x < Sh::NT; ++x) {
            const int d = 8 * x + 2 * t;
            const float2 y = unpack2(o[x][r]);
            if (d < dh) *reinterpret_cast<float2*>(dst + d) = make_float2(y.x * inv, y.y * inv);
        }
        if (splits > 1 && t == 0) { dst[dh] = r ? m1 : m0; dst[dh + 1] = L; }
    }
}

// One warp per (row, head) with more than one split: joins them in split order. Grid
// (rows, CTAs of 8 heads).
static __global__ void __launch_bounds__(256) paged_attn_join_kernel(const __grid_constant__ PagedAttnParams p) {
    const int lane = threadIdx.x & 31, row = blockIdx.x, h = blockIdx.y * 8 + (threadIdx.x >> 5), dh = p.c.dh;
    if (h >= p.H) return;
    int pos = 0;
    bool found = false;
    for (int base = 0; base < p.r.n_seq && !found; base += 32) {
        SeqRows q{0, 0, 0};
        if (base + lane < p.r.n_seq) q = seq_rows(p.r, base + lane);
        const unsigned m = __ballot_sync(0xffffffffu, row >= q.a && row < q.a + q.len);
        if (m) {
            pos = __shfl_sync(0xffffffffu, q.pos0() + row - q.a, __ffs(m) - 1);
            found = true;
        }
    }
    const int n = found ? row_splits(p, pos) : 0;
    if (n < 2) return;
    const int stride = dh + 4;
    const float* base = p.part + ((size_t)row * p.H + h) * p.nsplit * stride;
    float M = -INFINITY;
    for (int s = lane; s < n; s += 32) M = fmaxf(M, base[(size_t)s * stride + dh]);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float B = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int s = 0; s < n; ++s) {
        const float* ps = base + (size_t)s * stride;
        const float e = exp2_fast(ps[dh] - B);
        L = ffma(ps[dh + 1], e, L);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = 4 * lane + 128 * i;
            if (d >= dh) continue;
            const float4 x = *reinterpret_cast<const float4*>(ps + d);
            acc[i].x = ffma(x.x, e, acc[i].x); acc[i].y = ffma(x.y, e, acc[i].y);
            acc[i].z = ffma(x.z, e, acc[i].z); acc[i].w = ffma(x.w, e, acc[i].w);
        }
    }
    const float inv = L == 0.0f ? 0.0f : fdiv(1.0f, L);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = 4 * lane + 128 * i;
        if (d < dh)
            *reinterpret_cast<float4*>(p.out + (size_t)row * p.ldo + (size_t)h * dh + d) =
                make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
    }
}

}  // namespace b2
