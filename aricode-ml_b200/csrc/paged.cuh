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
struct PagedAttnParams {
    PagedKv c;
    PagedRows r;
    const float* q;          // [n_rows][ldq], rotated and pre-scaled
    float* out;              // [n_rows][ldo]
    long long ldq, ldo;
    int H;
    int* err;
};

// One warp per (row, head): 32 keys at a time, a lane per key for the scores, then
// the lanes over the head's elements for the sum.
static __global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
    __shared__ __align__(16) float qs[4][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dh = p.c.dh;
    const long long item = (long long)blockIdx.x * 4 + warp;
    if (item >= (long long)p.r.n_rows * p.H) return;
    const int row = (int)(item / p.H), h = (int)(item % p.H), kvh = h / (p.H / p.c.KVH);
    int s = -1, kv = 0, pos = -1;
    for (int base = 0; base < p.r.n_seq && s < 0; base += 32) {
        SeqRows q{0, 0, 0};
        if (base + lane < p.r.n_seq) q = seq_rows(p.r, base + lane);
        const unsigned m = __ballot_sync(0xffffffffu, row >= q.a && row < q.a + q.len);
        if (m) {
            const int src = __ffs(m) - 1;
            s = base + src;
            kv = __shfl_sync(0xffffffffu, q.kv, src);
            pos = __shfl_sync(0xffffffffu, q.pos0() + row - q.a, src);
        }
    }
    if (s < 0) return;                                             // behind the last sequence
    if (kv > p.r.cap && lane == 0) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
    for (int d = lane; d < dh; d += 32) qs[warp][d] = p.q[(size_t)row * p.ldq + (size_t)h * dh + d];
    __syncwarp();
    const int n = min(pos + 1, p.r.cap), psz = 1 << p.c.page_log2;
    float m = -INFINITY, l = 0.0f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.0f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float sc = -INFINITY, vs = 0.0f;
        long long at = -1;
        if (j < n) {
            const int page = page_of(p.c, p.r, s, j);
            if (page >= 0) {
                const size_t head = (size_t)page * p.c.KVH + kvh;
                const size_t cell = head * (psz / kKvBlock) + (j & (psz - 1)) / kKvBlock;
                at = (long long)((head * psz + (j & (psz - 1))) * dh);
                float a = 0.0f;
                for (int d = 0; d < dh; d += 4) {
                    const char4 w = *reinterpret_cast<const char4*>(p.c.k + at + d);
                    a = ffma((float)w.x, qs[warp][d], a);
                    a = ffma((float)w.y, qs[warp][d + 1], a);
                    a = ffma((float)w.z, qs[warp][d + 2], a);
                    a = ffma((float)w.w, qs[warp][d + 3], a);
                }
                sc = fmul(a, p.c.ks[cell]);
                vs = p.c.vs[cell];
            } else {
                set_err(p.err, B2_DEV_ERR_BAD_PAGE);
            }
        }
        float mx = sc;
        for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        mx = fmaxf(mx, m);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float e = at < 0 ? 0.0f : exp_f(fsub(sc, base));
        const float back = exp_f(fsub(m, base));
        m = mx;
        l = ffma(l, back, butterfly32(e));
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmul(o[i], back);
        const float w = at < 0 ? 0.0f : fmul(e, vs);
        for (int t = 0; t < min(32, n - j0); ++t) {
            const long long a = __shfl_sync(0xffffffffu, at, t);
            const float wt = __shfl_sync(0xffffffffu, w, t);
            if (a < 0) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = lane + 32 * i;
                if (d < dh) o[i] = ffma(wt, (float)p.c.v[a + d], o[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < dh) p.out[(size_t)row * p.ldo + (size_t)h * dh + d] = l == 0.0f ? 0.0f : fdiv(o[i], l);
    }
}

}  // namespace b2
