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
#include "umma.cuh"

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
    q.a = min(max(r.row_start[s], 0), r.n_rows);
    q.len = min(max(r.row_start[s + 1], q.a), r.n_rows) - q.a;
    q.kv = max(r.kv_len[s], 0);
    return q;
}

// page of position pos of sequence s, or -1
__device__ __forceinline__ int page_of(const PagedKv& c, const PagedRows& r, int s, int pos) {
    const int id = r.table[(size_t)s * r.max_pages + (pos >> c.page_log2)];
    return (unsigned)id < (unsigned)c.n_pages ? id : -1;
}

// Start of every kernel here: they are launched with programmatic serialisation, so that
// a launch comes up while the one before it drains, and read nothing before that is
// complete. The launch before it may have written what they read (rows, lengths, pages,
// codes, scales), within this one's lifetime: such loads are plain ones, which stay behind
// the wait; read-only loads (__ldg) are for gains and rotation tables alone. (Same times.)
__device__ __forceinline__ void after_previous() {
    pdl_launch_dependents();
    pdl_wait();
}

// Plain loads too, free to move among the shared-memory stores around them but not before
// the wait (the split kernel's codes: as C++ loads they cost <64, 8> 52 bytes of spills and
// 3 % of attend-long).
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8(const void* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// A run: the rows of one sequence that lie in one block of 16 tokens.
struct BlockRun {
    int s;          // sequence (-1: none)
    int row, n;     // its rows row .. row + n - 1 (1 <= n <= 16)
    int pos;        // position of the first one
};

// Run number `item` of the call, found by one warp: lanes count the runs of 32
// sequences at a time. Run 0 also checks all row ranges: only where a start is below the
// one before it can two overlap (and their runs be more than the grid covers).
__device__ __forceinline__ BlockRun find_run(const PagedRows& r, int item, int* err, int lane) {
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
            if (item == 0) {
                if (r.row_start[s + 1] < r.row_start[s]) set_err(err, B2_DEV_ERR_BAD_ROWS);
                if (q.len > 0 && q.kv > r.cap) set_err(err, B2_DEV_ERR_KV_OVERFLOW);
            }
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
    return out;
}

// ------------------------------------------------------------------ norm + rotation
// Head vectors in registers: LPH lanes hold a vector, VPL float4s each (lane l of
// the group the elements 4 l + 4 LPH i ..), so dh <= 4 LPH VPL.

// 1 / sqrt(mean x^2 + eps) of a vector (inv_dh = 1 / dh); rsqrtf is within 2^-22.9, no
// more than the sum's own roundings
template <int LPH, int VPL>
__device__ __forceinline__ float head_rms(const float4 (&x)[VPL], float inv_dh, float eps) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) a = ffma(x[i].x, x[i].x, ffma(x[i].y, x[i].y, ffma(x[i].z, x[i].z, ffma(x[i].w, x[i].w, a))));
#pragma unroll
    for (int o = LPH / 2; o >= 1; o >>= 1) a = fadd(a, __shfl_xor_sync(0xffffffffu, a, o));
    return rsqrtf(ffma(a, inv_dh, eps));
}

// The norm's gains and the rotation of two neighbouring pairs in one: the products of
// gain and (cos, sin) are made once for all vectors of a row, then a vector costs what
// the rotation alone would. Without gains this is b2_rope_apply's arithmetic.
struct Turn {
    float4 c, s;             // own and the other element's factor, signs in
};
__device__ __forceinline__ Turn make_turn(const float4& t, const float4& g) {
    Turn r;
    r.c = make_float4(fmul(g.x, t.x), fmul(g.y, t.x), fmul(g.z, t.z), fmul(g.w, t.z));
    r.s = make_float4(-fmul(g.y, t.y), fmul(g.x, t.y), -fmul(g.w, t.w), fmul(g.z, t.w));
    return r;
}
// b * s + a * c with two products and a sum, so that nothing depends on which is fused
__device__ __forceinline__ float4 turn4(const float4& x, const Turn& t) {
    return make_float4(fadd(fmul(x.x, t.c.x), fmul(x.y, t.s.x)), fadd(fmul(x.x, t.s.y), fmul(x.y, t.c.y)),
                       fadd(fmul(x.z, t.c.z), fmul(x.w, t.s.z)), fadd(fmul(x.z, t.s.w), fmul(x.w, t.c.w)));
}

struct NormRopeParams {
    const float* q;          // [n_rows][ldq], H heads side by side
    const float* k;          // [n_rows][ldk]
    float* qo;
    float* ko;
    long long ldq, ldk, ldqo, ldko;
    const float* gq;         // [dh] or nullptr: no norm
    const float* gk;
    float eps, q_scale, inv_dh;
    const float* table;      // [table_rows][dh] (cos, sin) pairs or nullptr: no rotation
    int table_rows;
    const int* pos;          // [n_rows]; negative: the row is left alone
    int n_rows, H, KVH, dh;
    int* err;
};

// HPU neighbouring vectors of one row's queries or keys (group number `grp` of them: H /
// HPU groups of queries, then the keys') through norm, rotation and scale, all loads
// first. `live`: the lane group has work (every lane of the warp runs along for the
// shuffles).
template <int LPH, int VPL, int HPU>
__device__ __forceinline__ void norm_rope_heads(const NormRopeParams& p, int row, int grp, int gl, bool live, int pos) {
    const int qgroups = (p.H + HPU - 1) / HPU;
    const bool isq = grp < qgroups;
    const int h0 = (isq ? grp : grp - qgroups) * HPU, cnt = live ? min((isq ? p.H : p.KVH) - h0, HPU) : 0;
    const float* src = (isq ? p.q + (size_t)row * p.ldq : p.k + (size_t)row * p.ldk) + (size_t)h0 * p.dh + 4 * gl;
    float* dst = (isq ? p.qo + (size_t)row * p.ldqo : p.ko + (size_t)row * p.ldko) + (size_t)h0 * p.dh + 4 * gl;
    float4 x[HPU][VPL];
#pragma unroll
    for (int u = 0; u < HPU; ++u)
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            x[u][i] = u < cnt && 4 * (gl + LPH * i) < p.dh ? *reinterpret_cast<const float4*>(src + u * p.dh + 4 * LPH * i)
                                                           : make_float4(0.f, 0.f, 0.f, 0.f);
    const float* g = isq ? p.gq : p.gk;
    Turn t[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int d = 4 * (gl + LPH * i);
        t[i] = make_turn(cnt > 0 && p.table && d < p.dh ? __ldg(reinterpret_cast<const float4*>(p.table + (size_t)pos * p.dh + d))
                                                        : make_float4(1.f, 0.f, 1.f, 0.f),
                         g && d < p.dh ? __ldg(reinterpret_cast<const float4*>(g + d)) : make_float4(1.f, 1.f, 1.f, 1.f));
    }
    const bool norm = p.gq || p.gk;                            // the same for the whole warp: it shuffles
    const float sc = isq ? p.q_scale : 1.0f;
#pragma unroll
    for (int u = 0; u < HPU; ++u) {
        float r = sc;
        if (norm) {
            const float m = head_rms<LPH, VPL>(x[u], p.inv_dh, p.eps);
            if (g) r = fmul(m, sc);
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            float4 y = turn4(x[u][i], t[i]);
            y = make_float4(fmul(y.x, r), fmul(y.y, r), fmul(y.z, r), fmul(y.w, r));
            if (u < cnt && 4 * (gl + LPH * i) < p.dh) *reinterpret_cast<float4*>(dst + u * p.dh + 4 * LPH * i) = y;
        }
    }
}

// One lane group per (row, HPU heads). Bound by memory once there are enough rows; what
// a vector costs in instructions comes next (see make_turn). 8191 rows of 40 heads of 128:
// 55 us, 6.2 TB/s, 0.94 of a plain copy's rate; a row of 36 heads of 64: 3.4 us.
template <int LPH, int VPL, int HPU>
__global__ void __launch_bounds__(256) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    after_previous();
    const unsigned per_row = (p.H + HPU - 1) / HPU + (p.KVH + HPU - 1) / HPU;
    const unsigned unit = (blockIdx.x * 256u + threadIdx.x) / LPH, row = unit / per_row;
    const int gl = threadIdx.x % LPH;
    bool live = row < (unsigned)p.n_rows;
    int pos = 0;
    if (live && p.pos) {
        pos = p.pos[row];
        if (pos < 0) live = false;
        else if (p.table && pos >= p.table_rows) {
            live = false;
            set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
        }
    }
    norm_rope_heads<LPH, VPL, HPU>(p, live ? (int)row : 0, (int)(unit % per_row), gl, live, live ? pos : 0);
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

// The run's rows of one head's K or V by WPT warps (this one is number `part`, `top` a
// word of theirs in shared memory, 0): NP passes of WPT * 32 / LPH rows in registers. The
// block's new scale is known when all rows have been seen; if they are more than the
// registers hold (WPT = 1) they are fetched again for the codes.
template <int LPH, int VPL, int NP, int WPT>
__device__ __forceinline__ void append_head(const AppendParams& p, const BlockRun& run, int page, int head, bool is_k,
                                            int lane, int part, unsigned* top) {
    constexpr int RPW = 32 / LPH * WPT;            // rows per pass
    const int dh = p.c.dh, gl = lane % LPH, g = part * (32 / LPH) + lane / LPH;
    const float* src = (is_k ? p.k : p.v) + (size_t)head * dh;
    const long long ld = is_k ? p.ldk : p.ldv;
    const bool rope = is_k && p.nr.table;
    const int psz = 1 << p.c.page_log2;
    const int off = run.pos & (psz - 1), o0 = run.pos % kKvBlock;
    const size_t cell = ((size_t)page * p.c.KVH + head) * (psz / kKvBlock) + off / kKvBlock;
    float* sp = (is_k ? p.c.ks : p.c.vs) + cell;
    int8_t* codes = (is_k ? p.c.k : p.c.v) + cell * kKvBlock * dh;    // the block's 16 rows
    // a block that starts with this run has no older rows: its scale starts afresh
    const float old = o0 == 0 ? 0.0f : *sp;
    float4 x[NP][VPL];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int i = i0 + j * RPW + g;
#pragma unroll
            for (int e = 0; e < VPL; ++e) {
                const int d = 4 * (gl + LPH * e);
                x[j][e] = (i < run.n && d < dh) ? *reinterpret_cast<const float4*>(src + (size_t)(run.row + i) * ld + d)
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
            for (int j = 0; j < NP; ++j) {
                if (i0 + j * RPW >= run.n) continue;
                // (rows past the run are zeros and stay so: without an eps their norm is not a number)
                const float rms = head_rms<LPH, VPL>(x[j], p.nr.inv_dh, p.nr.eps), r = i0 + j * RPW + g < run.n ? rms : 0.0f;
#pragma unroll
                for (int e = 0; e < VPL; ++e)
                    x[j][e] = make_float4(fmul(fmul(x[j][e].x, r), gv[e].x), fmul(fmul(x[j][e].y, r), gv[e].y),
                                          fmul(fmul(x[j][e].z, r), gv[e].z), fmul(fmul(x[j][e].w, r), gv[e].w));
            }
        }
        if (rope) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int i = i0 + j * RPW + g;
#pragma unroll
                for (int e = 0; e < VPL; ++e) {
                    const int d = 4 * (gl + LPH * e);
                    if (i < run.n && d < dh)
                        x[j][e] = turn4(x[j][e], make_turn(__ldg(reinterpret_cast<const float4*>(p.nr.table + (size_t)(run.pos + i) * dh + d)),
                                                           make_float4(1.f, 1.f, 1.f, 1.f)));
                }
            }
        }
    };
    unsigned am = 0u;                              // largest |x| as bits: a NaN or infinity is above 0x7f7fffff
    for (int i0 = 0; i0 < (NP * RPW < kKvBlock ? run.n : 1); i0 += NP * RPW) {
        fetch(i0);
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int e = 0; e < VPL; ++e)
                am = max(am, max(max(__float_as_uint(x[j][e].x) & 0x7fffffffu, __float_as_uint(x[j][e].y) & 0x7fffffffu),
                                 max(__float_as_uint(x[j][e].z) & 0x7fffffffu, __float_as_uint(x[j][e].w) & 0x7fffffffu)));
    }
    am = __reduce_max_sync(0xffffffffu, am);
    if constexpr (WPT > 1) {
        if (lane == 0) atomicMax(top, am);
        __syncthreads();                           // also: every warp has read the old scale
        am = *top;
    }
    float now = am >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fdiv(__uint_as_float(am), 127.0f);
    if (!(now <= old)) {                           // grown (or NaN on either side)
        if (old != old) now = old;
        else if (now == now && o0 > 0) {           // older rows to the new scale
            const float ratio = fdiv(old, now);
            for (int b = (part * 32 + lane) * 4; b < o0 * dh; b += 128 * WPT) {
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
    if (lane == 0 && part == 0) *sp = now;
    // x / now rounded to an integer: the quotient by the reciprocal and one correction is
    // the f32 division's (a scale whose reciprocal or remainders could leave f32's normal
    // range takes the division itself); adding 1.5 * 2^23 rounds it into the low byte
    const bool some = now > 0.0f;                  // false for a block of zeros and for a NaN scale
    const bool plain = now > 0x1p-100f && now < 0x1p100f;
    const float inv = fdiv(1.0f, now);
    auto code = [&](float v) {
        float q;
        if (plain) {
            q = fmul(v, inv);
            q = ffma(ffma(-q, now, v), inv, q);
        } else {
            q = some ? fmaxf(-127.0f, fminf(127.0f, fdiv(v, now))) : 0.0f;
        }
        return __float_as_uint(fadd(q, 12582912.0f));
    };
    for (int i0 = 0; i0 < (NP * RPW < kKvBlock ? run.n : 1); i0 += NP * RPW) {
        if constexpr (NP * RPW < kKvBlock)
            if (run.n > NP * RPW) fetch(i0);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int i = i0 + j * RPW + g;
#pragma unroll
            for (int e = 0; e < VPL; ++e) {
                const int d = 4 * (gl + LPH * e);
                const uint32_t lo = __byte_perm(code(x[j][e].x), code(x[j][e].y), 0x0040),
                               hi = __byte_perm(code(x[j][e].z), code(x[j][e].w), 0x0040);
                if (i < run.n && d < dh)
                    *reinterpret_cast<uint32_t*>(codes + (size_t)(o0 + i) * dh + d) = __byte_perm(lo, hi, 0x5410);
            }
        }
    }
}

// the run of this CTA without the rows that lie past the table (they have no rotation)
__device__ __forceinline__ BlockRun run_in_table(const AppendParams& p, int lane) {
    BlockRun run = find_run(p.r, blockIdx.x, p.err, lane);
    if (run.s >= 0 && p.nr.table && run.pos + run.n > p.nr.table_rows) {
        if (lane == 0) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
        run.n = max(p.nr.table_rows - run.pos, 0);
    }
    return run;
}

// a run's queries, HPU vectors of a row at a time: unit numbers from `unit` on
template <int LPH, int VPL, int HPU>
__device__ __forceinline__ void append_queries(const AppendParams& p, const BlockRun& run, int unit, int step, int lane) {
    const int per_row = (p.nr.H + HPU - 1) / HPU, units = run.n * per_row;
    for (int first = unit - lane / LPH; first < units; first += step, unit += step) {   // whole warps
        const int i = unit / per_row;
        const bool live = unit < units;
        norm_rope_heads<LPH, VPL, HPU>(p.nr, live ? run.row + i : 0, unit % per_row, lane % LPH, live,
                                       live ? run.pos + i : 0);
    }
}

// Grid (runs, CTAs of a run): every warp finds the run; WPT warps of the first kv_ctas
// take one head's K or V of it, those of the others queries.
// WPT = 1, NP = 1: for calls of single rows. WPT = 4: up to 16 rows; with one warp holding
// all of them (120 registers, 16 warps an SM) 6300 rows took 41 us. Few registers, so
// that many runs are on the SMs at once: it is bound by the latency of run -> page ->
// scale and older codes. 6300 rows of 8 heads of 128: 27 to 29 us; 64 single rows of 32: 8 us.
// Six CTAs an SM for d_head 65 to 128 instead of the five that its registers allow: 148 ->
// 144 us for 6300 rows of 32 + 32 heads with queries and read back; at 64 no difference.
template <int LPH, int VPL, int NP, int WPT>
__global__ void __launch_bounds__(256, WPT == 4 && LPH == 32 && VPL == 1 ? 6 : 1) kv_append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ unsigned top[8 / WPT];
    after_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if constexpr (WPT > 1) {
        if (threadIdx.x < 8 / WPT) top[threadIdx.x] = 0u;
        __syncthreads();
    }
    const BlockRun run = run_in_table(p, lane);
    if (run.s < 0 || run.n == 0) return;
    if ((int)blockIdx.y < p.kv_ctas) {
        const int task = (blockIdx.y * 8 + warp) / WPT;        // (WPT = 4: two tasks a CTA, K and V of a head)
        if (task >= 2 * p.c.KVH) return;
        const int page = page_of(p.c, p.r, run.s, run.pos);
        if (page < 0) {
            if (lane == 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
            return;
        }
        append_head<LPH, VPL, NP, WPT>(p, run, page, task >> 1, (task & 1) == 0, lane, warp % WPT, top + warp / WPT);
        return;
    }
    append_queries<LPH, VPL, 1>(p, run, ((blockIdx.y - p.kv_ctas) * 256 + threadIdx.x) / LPH,
                                (gridDim.y - p.kv_ctas) * 256 / LPH, lane);
}

// the queries of long calls, in a launch of their own: the registers that hold a block's
// rows above would leave them too few warps to keep the memory busy (6300 rows of 32
// heads of 128: 33 us, 6.2 TB/s)
template <int LPH, int VPL>
__global__ void __launch_bounds__(256) append_queries_kernel(const __grid_constant__ AppendParams p) {
    after_previous();
    const BlockRun run = run_in_table(p, threadIdx.x & 31);
    if (run.s < 0) return;
    append_queries<LPH, VPL, 4>(p, run, (blockIdx.y * 256 + threadIdx.x) / LPH, gridDim.y * 256 / LPH, threadIdx.x & 31);
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
// (contiguous bytes) into values, LPR lanes a row of 8 codes each, all loads first.
// Bound by memory (13.9 K rows of 32 heads to bf16: 56 us, 0.89 of a plain copy's rate).
// Rows on a missing page become zeros.
template <bool BF16, int LPR>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ ReadParams p) {
    after_previous();
    constexpr int RPP = 32 / LPR, NP = kKvBlock / RPP;         // rows a pass, passes
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const BlockRun run = find_run(p.r, blockIdx.x, p.err, lane);
    if (run.s < 0) return;
    const int task = blockIdx.y * 8 + warp;
    if (task >= 2 * p.c.KVH) return;
    const int head = task >> 1, dh = p.c.dh, d = 8 * (lane % LPR), r0 = lane / LPR;
    const bool is_k = (task & 1) == 0;
    const int page = page_of(p.c, p.r, run.s, run.pos);
    if (page < 0 && lane == 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
    const int psz = 1 << p.c.page_log2;
    const size_t cell = ((size_t)max(page, 0) * p.c.KVH + head) * (psz / kKvBlock) + (run.pos & (psz - 1)) / kKvBlock;
    const float s = page < 0 ? 0.0f : (is_k ? p.c.ks : p.c.vs)[cell];
    const int8_t* codes = (is_k ? p.c.k : p.c.v) + (cell * kKvBlock + run.pos % kKvBlock) * dh + d;
    uint2 w[NP];
#pragma unroll
    for (int x = 0; x < NP; ++x) {
        const int r = x * RPP + r0;
        w[x] = page >= 0 && r < run.n && d < dh ? *reinterpret_cast<const uint2*>(codes + r * dh) : make_uint2(0u, 0u);
    }
    const size_t at = (size_t)run.row * p.ld + (size_t)head * dh + d;
#pragma unroll
    for (int x = 0; x < NP; ++x) {
        const int r = x * RPP + r0;
        if (r >= run.n || d >= dh) continue;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = fmul((float)(signed char)(w[x].x >> (8 * e)), s);
            f[4 + e] = fmul((float)(signed char)(w[x].y >> (8 * e)), s);
        }
        if constexpr (BF16) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_k ? p.k : p.v) + at + r * p.ld) =
                make_uint4(bf16x2_bits(f[0], f[1]), bf16x2_bits(f[2], f[3]), bf16x2_bits(f[4], f[5]), bf16x2_bits(f[6], f[7]));
        } else {
            float* o = static_cast<float*>(is_k ? p.k : p.v) + at + r * p.ld;
            *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
}

// ------------------------------------------------------------------ attention
// The codes are exact small integers, so both products run as integer dots on the
// tensor cores (warp-level s8 MMAs) with the f32 side split into three signed
// base-256 digits: X = rint(x 2^..) with |X| <= kDigitMax = d2 65536 + d1 256 + d0,
// 23 bits below the row's largest element. (That loses bits of the others where one
// channel stands out, but with keys in 8 bits they hardly count: the rounding moves a score
// by at most 2^-24 max|q| sum|k| <= 2^-24 127 d_head max|q| scale, the cache's own rounding of
// the largest channel by up to max|q| scale / 2. The same holds for weights and values. A
// fourth digit would need 16 KB of the tcgen05 kernel's shared memory, where 9 KB are left.)
// The digit sums are exact in int32 and are joined in f32, so a score or an output carries
// the error of one 23-bit rounding per factor instead of a chain of f32 roundings, at a
// third of the int8 rate and without converting a single code.
// Three digits in [-128, 127] reach 2^23 - 1 - 0x8080 = 8355711; a little below it,
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

// d2 65536 + d1 256 + d0 of two neighbouring sums a, b: the lower two digits joined as
// integers (256 products: below 2^30)
__device__ __forceinline__ f32x2 join_digits(int a2, int b2, int a1, int b1, int a0, int b0) {
    return fma2(pack2((float)a2, (float)b2), pack2(65536.0f, 65536.0f), pack2((float)(a1 * 256 + a0), (float)(b1 * 256 + b0)));
}
__device__ __forceinline__ f32x2 join_digits(const int (&c)[3][4], int y) {
    return join_digits(c[2][y], c[2][y + 1], c[1][y], c[1][y + 1], c[0][y], c[0][y + 1]);
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

// the same for weights, whose largest is a probability times a value scale: the
// approximate reciprocal is within 2^-22, and kDigitMax leaves room for that
__device__ __forceinline__ float weight_factor(float top) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(top));
    return fminf(r * (float)kDigitMax, 0x1p126f);
}
__device__ __forceinline__ float weight_unit(float f) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(f));
    return r;
}

struct PagedAttnParams {
    PagedKv c;
    PagedRows r;
    const float* q;          // [n_rows][ldq], rotated and pre-scaled
    float* out;              // [n_rows][ldo]
    long long ldq, ldo;
    int H, G;                // G = H / KVH
    int lo, hi;              // columns (rows * G) of the sequences that this launch takes
    int kc_log2;             // keys per split of this launch's sequences
    int few;                 // sequences of up to `few` columns have splits of
    int kc_few, kc_many;     // 2^kc_few keys, the others of 2^kc_many
    int join_rows;           // 0: every row may have splits; else only the first join_rows
                             // of each sequence of up to `few` columns
    // Partial results [slot][H][nsplit][dh + 4]: o, m (base 2), l; an area for each kind. A
    // slot is a row; in the few-row kind's area with few_rows > 0 it is the row's number in
    // its sequence, of few_rows a sequence. nsplit: splits of cap keys
    int few_rows, nsplit_few, nsplit_many;
    float* part_few;
    float* part_many;
    int* err;
};

// A unit of attention work: columns col0 .. of one KV head's (row, head) pairs of a
// sequence, against keys of split `split`.
struct AttnItem {
    int s, a, len, kv;       // sequence and its rows (s < 0: none left)
    int kvh, tile, split;
};

// splits of n keys (at least one: it also writes rows that see none)
__device__ __forceinline__ int splits_of(int kc_log2, int n) { return max((n + (1 << kc_log2) - 1) >> kc_log2, 1); }

// Most items of one sequence (the host refuses calls that could have more): the sums
// over 32 lanes stay in 32 bits whatever the row ranges are.
constexpr int kMaxItems = 1 << 26;

// Item number `item` of the call (tiles of NC rows), found by one warp. OneWord: s becomes
// sequence * 1024 + KV head (up to 2^16 and 2^10 of them) and kvh stays 0, for the split
// kernel, which has no register left for both.
template <int NC, bool OneWord = false>
__device__ __forceinline__ AttnItem find_item(const PagedAttnParams& p, unsigned item, int lane) {
    AttnItem out{-1, 0, 0, 0, 0, 0, 0};
    unsigned before = 0;
    for (int base = 0; base < p.r.n_seq && before < (1u << 31); base += 32) {
        const int s = base + lane;
        SeqRows q{0, 0, 0};
        unsigned cnt = 0;
        int tiles = 0;
        if (s < p.r.n_seq) {
            q = seq_rows(p.r, s);
            const long long cols = (long long)q.len * p.G;
            if (q.len > 0 && cols >= p.lo && cols <= p.hi) {
                if (q.kv > p.r.cap) set_err(p.err, B2_DEV_ERR_KV_OVERFLOW);
                tiles = (q.len * p.G + NC - 1) / NC;
                cnt = (unsigned)min((long long)tiles * p.c.KVH * splits_of(p.kc_log2, min(q.kv, p.r.cap)), (long long)kMaxItems);
            }
        }
        const unsigned total = __reduce_add_sync(0xffffffffu, cnt);
        if (item - before < total) {
            unsigned incl = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const int src = __ffs(__ballot_sync(0xffffffffu, incl > item - before)) - 1;
            const unsigned idx = item - before - __shfl_sync(0xffffffffu, incl - cnt, src);
            out.s = base + src;
            out.a = __shfl_sync(0xffffffffu, q.a, src);
            out.len = __shfl_sync(0xffffffffu, q.len, src);
            out.kv = __shfl_sync(0xffffffffu, q.kv, src);
            // the last rows first: with causal lengths they are the longest
            const unsigned splits = splits_of(p.kc_log2, min(out.kv, p.r.cap)), rest = idx / (unsigned)p.c.KVH;
            const int kvh = (int)(idx % (unsigned)p.c.KVH);
            if constexpr (OneWord) out.s = out.s * 1024 + kvh;
            else out.kvh = kvh;
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
    return splits_of(p.kc_log2, min(pos + 1, p.r.cap));
}

// partial result `split` of head h of row tok of sequence s (row `row` of the call)
__device__ __forceinline__ float* few_part(const PagedAttnParams& p, int s, int tok, int row, int h, int split) {
    const size_t slot = p.few_rows ? (size_t)s * p.few_rows + tok : (size_t)row;
    return p.part_few + ((slot * p.H + h) * p.nsplit_few + split) * (p.c.dh + 4);
}
__device__ __forceinline__ float* many_part(const PagedAttnParams& p, int row, int h, int split) {
    return p.part_many + (((size_t)row * p.H + h) * p.nsplit_many + split) * (p.c.dh + 4);
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
        x[i] = (live && d < dh) ? *reinterpret_cast<const float4*>(qr + d) : make_float4(0.f, 0.f, 0.f, 0.f);
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
// go from global memory straight into B fragments (keys as they lie; values turned by
// byte permutes inside a thread), nothing is staged. A step's keys are requested when
// the previous step's scores are done, its values when the previous step's output is,
// across items too: each CTA runs through its items with the next item's place, pages,
// scales and queries fetched one item ahead, so a warp always has loads in flight.
// A = digits: a 16-row tile holds digit 2 of the 8 columns above digit 1, a second one
// digit 0, so that a thread gets all three digit sums of its (column, key) pairs. The
// second one's rows 8 to 15 hold the digits of the other 16 elements of each part: of
// its two products one counts in the upper, one in the lower half.
// The four warps' (m, l, o) meet in shared memory, one barrier an item.
constexpr int kSplitWarps = 4;
constexpr int kSplitCols = 8;
// (at most 512 keys a split: its blocks are one a lane)

// NC columns an item: 8, or 2 for calls of one or two columns a KV head (decode without
// shared heads). Then the digits are the MMA's columns instead: A = codes (16 keys x d,
// 16 elements x keys), column 4 c + e = digit e of head column c, and every digit column
// keeps its own f32 output until the end: a quarter of the MMAs and half of the folding.
template <int DP, int NC>
struct SplitShape {
    static constexpr int NH = DP / 64;             // 64-byte parts of a key row
    static constexpr int VW = DP / 32;             // 32-bit words of a value row that a lane holds
    static constexpr int NT = DP / 8;              // output tiles of 8 elements
    static constexpr int QBytes = NH * (NC == 8 ? 3 : 1) * 32 * 16;        // A fragments [part][hi, hi, lo][lane]; B [part][lane]
    static constexpr int WBytes = NC == 8 ? 0 : kSplitWarps * 2 * 32 * 4;  // narrow: a step's weights [warp][column][key]
    static constexpr int MergeBytes = kSplitWarps * NC * (DP + 4) * 4;
    static constexpr int Smem = 2 * (QBytes + 32 + MergeBytes) + WBytes;
};

struct SplitItem {
    AttnItem it;             // its sequence and KV head in one word
    __device__ __forceinline__ int seq() const { return it.s >> 10; }
    __device__ __forceinline__ int kvh() const { return it.s & 1023; }
    int cols, col0, n, j0, jend;
    int cell;                // block `lane` of the split in the pool (codes start at 16 dh
    float ks, vs;            // times that; -1: page outside the pool, -2: past the end), scales
};

// the CTA's next item from number `item` on (stride gridDim.x) that has keys to look at
template <int NC>
__device__ __forceinline__ SplitItem next_split_item(const PagedAttnParams& p, unsigned& item, int lane) {
    SplitItem w;
    for (;; item += gridDim.x) {
        w.it = find_item<NC, true>(p, item, lane);
        w.cell = -2;
        if (w.it.s < 0) return w;
        w.col0 = w.it.tile * NC;
        w.cols = min(w.it.len * p.G - w.col0, NC);
        const int last = w.it.len == 1 ? 0 : (w.col0 + w.cols - 1) / p.G;  // the tile's last token
        w.n = min(w.it.kv - w.it.len + last + 1, p.r.cap);
        w.j0 = w.it.split << p.kc_log2;
        if (w.j0 < w.n || w.it.split == 0) break;                          // else the tile ends before this split
    }
    w.jend = min(w.n, w.j0 + (1 << p.kc_log2));
    const int j = w.j0 + 16 * lane;
    w.ks = w.vs = 0.0f;
    if (j < w.jend) {
        const int page = page_of(p.c, p.r, w.seq(), j), b = p.c.page_log2 - 4;
        w.cell = page < 0 ? -1 : ((page * p.c.KVH + w.kvh()) << b) + ((j >> 4) & ((1 << b) - 1));
        if (page < 0) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
        else { w.ks = p.c.ks[w.cell]; w.vs = p.c.vs[w.cell]; }
    }
    return w;
}

// 64 sequences x 1152 keys, 32 heads of 128 (NC = 2): 118 us with the join, 5.1 TB/s; 42 %
// of the issue slots, the longest stall is on the codes' loads. With 4 CTAs an SM it
// spills at 128 registers: 160 us.
template <int DP, int NC>
__global__ void __launch_bounds__(kSplitWarps * 32, DP == 256 ? 2 : DP == 128 ? 3 : 4)
paged_attn_split_kernel(const __grid_constant__ PagedAttnParams p) {
    using Sh = SplitShape<DP, NC>;
    constexpr bool kNarrow = NC == 2;
    extern __shared__ __align__(16) unsigned char ps_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int dh = p.c.dh;
    after_previous();
    unsigned item = blockIdx.x;
    SplitItem cur = next_split_item<NC>(p, item, lane);
    if (cur.it.s < 0) return;

    uint4 kf[4][Sh::NH];                                                   // a step's keys 8 x + g
    uint32_t vf[2][4][Sh::VW];                                             // its values: [block][key][words], keys 2t + {0, 1, 8, 9},
                                                                           // narrow 4t + {0, 1, 2, 3}
    // Blocks that are not there and elements past dh are read from the pool's first block and
    // row: they meet masked weights and zero digits, or make elements that are not stored.
    int kd[Sh::NH], vd[(Sh::VW + 3) / 4];                                  // element offsets inside a row
#pragma unroll
    for (int h = 0; h < Sh::NH; ++h) kd[h] = 64 * h + 16 * t < dh ? 64 * h + 16 * t : 0;
#pragma unroll
    for (int u = 0; u < (Sh::VW + 3) / 4; ++u) vd[u] = (DP / 8) * g + 16 * u < dh ? (DP / 8) * g + 16 * u : 0;
    auto load_keys = [&](int c0, int c1) {
        c0 = max(c0, 0); c1 = max(c1, 0);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int8_t* kr = p.c.k + ((long long)(x < 2 ? c0 : c1) * kKvBlock + 8 * (x & 1) + g) * dh;
#pragma unroll
            for (int h = 0; h < Sh::NH; ++h) kf[x][h] = load16(kr + kd[h]);
        }
    };
    auto load_values = [&](int c0, int c1) {
        c0 = max(c0, 0); c1 = max(c1, 0);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int8_t* vr = p.c.v + ((long long)(b ? c1 : c0) * kKvBlock + (kNarrow ? 4 : 2) * t) * dh;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int8_t* v = vr + (kNarrow ? i : (i & 1) + 8 * (i >> 1)) * dh;
                if constexpr (Sh::VW == 2) {
                    const uint2 x = load8(v + vd[0]);
                    vf[b][i][0] = x.x; vf[b][i][1] = x.y;
                } else {
#pragma unroll
                    for (int u = 0; u < Sh::VW / 4; ++u) {
                        const uint4 x = load16(v + vd[u]);
                        vf[b][i][4 * u] = x.x; vf[b][i][4 * u + 1] = x.y; vf[b][i][4 * u + 2] = x.z; vf[b][i][4 * u + 3] = x.w;
                    }
                }
            }
        }
    };
    // an item's queries as fragments in half `b` of the shared memory; 16 lanes a column
    auto put_queries = [&](const SplitItem& w, int b) {
        if (kNarrow && warp != kSplitWarps - 1) return;                    // two columns: the last warp's lanes
        unsigned char* qd = ps_raw + b * (Sh::QBytes + 32);
        const int col = kNarrow ? lane >> 4 : tid >> 4, cc = w.col0 + col, tok = w.it.len == 1 ? 0 : cc / p.G;
        query_digits<DP>(p.q + (size_t)(w.it.a + tok) * p.ldq + (size_t)(w.kvh() * p.G + cc - tok * p.G) * dh, col < w.cols, dh,
                         tid & 15, [&](int e, int d, uint32_t x) {
                             // words of the part's 16-byte unit: x, y make step 0, z, w step 1
                             const int h = d >> 6, q = (d >> 4) & 3, word = (d >> 2) & 3;
                             if constexpr (kNarrow) {
                                 *reinterpret_cast<uint32_t*>(qd + (h * 32 + 4 * (4 * col + e) + q) * 16 + 4 * word) = x;
                                 return;
                             }
                             const int frag = e ? word >> 1 : 2, reg = e ? 2 * (word & 1) + 2 - e : 2 * (word & 1) + (word >> 1);
                             *reinterpret_cast<uint32_t*>(qd + ((h * 3 + frag) * 32 + 4 * col + q) * 16 + 4 * reg) = x;
                         }, reinterpret_cast<float*>(qd + Sh::QBytes) + col);
    };

    int a0 = __shfl_sync(0xffffffffu, cur.cell, 2 * warp), a1 = __shfl_sync(0xffffffffu, cur.cell, 2 * warp + 1);
    load_keys(a0, a1);
    load_values(a0, a1);
    if constexpr (kNarrow)                                                 // columns 3 and 7 stay zero
        for (int i = tid; i < Sh::NH * 64; i += kSplitWarps * 32)
            *reinterpret_cast<uint32_t*>(ps_raw + (i & 1) * (Sh::QBytes + 32) + ((i >> 6) * 32 + 16 * ((i >> 5) & 1) + 12) * 16 +
                                         4 * ((i >> 1) & 15)) = 0u;
    put_queries(cur, 0);
    __syncthreads();
    for (int buf = 0;; buf ^= 1) {
        const unsigned char* qd = ps_raw + buf * (Sh::QBytes + 32);
        const int col = kNarrow ? t >> 1 : g;                              // the column of this lane's scores
        const float sqg = reinterpret_cast<const float*>(qd + Sh::QBytes)[col];   // their unit
        const int pos0 = cur.it.kv - cur.it.len;
        const int lim = col < cur.cols ? min(pos0 + (cur.it.len == 1 ? 0 : (cur.col0 + col) / p.G) + 1, cur.n) : 0;   // keys it sees
        // up to here no column needs a mask (idle columns have zero digits and no output)
        const int whole_end = __reduce_min_sync(0xffffffffu, col < cur.cols ? lim : cur.n);
        uint4 qb[Sh::NH];                                                  // narrow: the B fragments of column g's digit
        if constexpr (kNarrow)
#pragma unroll
            for (int h = 0; h < Sh::NH; ++h) qb[h] = reinterpret_cast<const uint4*>(qd)[h * 32 + lane];
        item += gridDim.x;
        SplitItem nxt = next_split_item<NC>(p, item, lane);
        if (kNarrow && nxt.it.s >= 0) put_queries(nxt, buf ^ 1);           // (its last readers are past their barrier)

        float m = -INFINITY;
        f32x2 l2 = 0ull;                                                   // this lane's part of the sum
        // wide: tile x: elements (DP/4) t + x, + DP/8 of column g; narrow: element (DP/8) g + x
        // of digit columns 2t, 2t + 1
        f32x2 o[Sh::NT];
#pragma unroll
        for (int x = 0; x < Sh::NT; ++x) o[x] = 0ull;

        int j = cur.j0 + warp * 32;
#pragma unroll 1
        do {                                                               // at least one step, if an empty one
            const int blk = (j - cur.j0) >> 4;
            const bool last = j + kSplitWarps * 32 >= cur.jend;
            // the next step's blocks, of the next item after the last one
            const int nblk = last ? 2 * warp : blk + 2 * kSplitWarps, ncell = last ? nxt.cell : cur.cell;
            const int na0 = __shfl_sync(0xffffffffu, ncell, nblk), na1 = __shfl_sync(0xffffffffu, ncell, nblk + 1);
            const float k0 = __shfl_sync(0xffffffffu, cur.ks, blk), k1 = __shfl_sync(0xffffffffu, cur.ks, blk + 1);
            const float v0 = __shfl_sync(0xffffffffu, cur.vs, blk), v1 = __shfl_sync(0xffffffffu, cur.vs, blk + 1);
            // scores (base 2): keys 8 x + 2t, + 1 for column g; narrow: keys 16 x + g, + 8 for column t / 2
            constexpr int NS = kNarrow ? 2 : 4;
            float2 s[NS];
            if constexpr (kNarrow) {
                const float up = t & 1 ? 65536.0f : 1.0f;                  // odd lanes have digit 2, even ones 0 and 1
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    int c[4];
#pragma unroll
                    for (int h = 0; h < Sh::NH; ++h) {
                        const uint4 k0 = kf[2 * x][h], k8 = kf[2 * x + 1][h];
                        if (h == 0) mma_s8_first(c, k0.x, k8.x, k0.y, k8.y, qb[h].x, qb[h].y);
                        else mma_s8(c, k0.x, k8.x, k0.y, k8.y, qb[h].x, qb[h].y);
                        mma_s8(c, k0.z, k8.z, k0.w, k8.w, qb[h].z, qb[h].w);
                    }
                    const float u = sqg * (x ? k1 : k0) * up;
                    s[x] = unpack2(mul2(pack2((float)(c[1] * 256 + c[0]), (float)(c[3] * 256 + c[2])), pack2(u, u)));
                    s[x].x += __shfl_xor_sync(0xffffffffu, s[x].x, 1);
                    s[x].y += __shfl_xor_sync(0xffffffffu, s[x].y, 1);
                }
            } else {
                int hi[4][4], lo[4][2][4];                                 // hi: digit 2 in 0, 1 and digit 1 in 2, 3
#pragma unroll
                for (int h = 0; h < Sh::NH; ++h) {
                    const uint4* fr = reinterpret_cast<const uint4*>(qd) + h * 96 + lane;
                    const uint4 f0 = fr[0], f1 = fr[32], f2 = fr[64];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if (h == 0) {
                            mma_s8_first(hi[x], f0.x, f0.y, f0.z, f0.w, kf[x][h].x, kf[x][h].y);
                            mma_s8_first(lo[x][0], f2.x, f2.y, f2.z, f2.w, kf[x][h].x, kf[x][h].y);
                            mma_s8_first(lo[x][1], f2.x, f2.y, f2.z, f2.w, kf[x][h].z, kf[x][h].w);
                        } else {
                            mma_s8(hi[x], f0.x, f0.y, f0.z, f0.w, kf[x][h].x, kf[x][h].y);
                            mma_s8(lo[x][0], f2.x, f2.y, f2.z, f2.w, kf[x][h].x, kf[x][h].y);
                            mma_s8(lo[x][1], f2.x, f2.y, f2.z, f2.w, kf[x][h].z, kf[x][h].w);
                        }
                        mma_s8(hi[x], f1.x, f1.y, f1.z, f1.w, kf[x][h].z, kf[x][h].w);
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float u = sqg * (x < 2 ? k0 : k1);
                    s[x] = unpack2(mul2(join_digits(hi[x][0], hi[x][1], hi[x][2], hi[x][3], lo[x][0][0] + lo[x][1][2],
                                                    lo[x][0][1] + lo[x][1][3]), pack2(u, u)));
                }
            }
            load_keys(na0, na1);
            const bool whole = j + 32 <= whole_end && (a0 | a1) >= 0 && v0 + v1 == v0 + v1;
            if (!whole) {
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const int key = kNarrow ? j + 16 * x + g : j + 8 * x + 2 * t, lx = (x < NS / 2 ? a0 : a1) >= 0 ? lim : 0;
                    if (key >= lx) s[x].x = -INFINITY;
                    if (key + (kNarrow ? 8 : 1) >= lx) s[x].y = -INFINITY;
                }
            }
            // over the lanes that hold a column's keys
            auto lanes_max = [](float v) {
                if constexpr (kNarrow) {
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                } else {
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                }
            };
            float mx = m;
#pragma unroll
            for (int x = 0; x < NS; ++x) mx = fmaxf(mx, fmaxf(s[x].x, s[x].y));
            mx = lanes_max(mx);
            const float base = mx == -INFINITY ? 0.0f : mx;
            const float back = exp2_fast(m - base);
            m = mx;
            f32x2 ls = 0ull;
            float2 e[NS];
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                e[x] = make_float2(exp2_fast(s[x].x - base), exp2_fast(s[x].y - base));
                ls = add2(ls, pack2(e[x].x, e[x].y));
                const float sv = x < NS / 2 ? v0 : v1;
                e[x] = unpack2(mul2(pack2(e[x].x, e[x].y), pack2(sv, sv)));
            }
            l2 = fma2(l2, pack2(back, back), ls);
            // weights p v_scale; a masked key weighs nothing even where the scale is NaN. A
            // score that is not a number has made the sum NaN, which is enough
            bool bad = false;
            if (!whole) {
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    if (s[x].x == -INFINITY) e[x].x = 0.0f;
                    if (s[x].y == -INFINITY) e[x].y = 0.0f;
                    bad |= e[x].x != e[x].x || e[x].y != e[x].y;
                }
            }
            float wt = bad ? INFINITY : 0.0f;
#pragma unroll
            for (int x = 0; x < NS; ++x) wt = fmaxf(wt, fmaxf(e[x].x, e[x].y));
            wt = lanes_max(wt);
            const float f = weight_factor(wt), u = wt < INFINITY ? weight_unit(f) : __int_as_float(0x7fffffff);
            if constexpr (kNarrow) {
                // weights to the lanes of their digit: column g = 4 c + e takes digit e of column
                // c's keys 4t .. 4t + 3 of each block
                uint32_t* wx = reinterpret_cast<uint32_t*>(ps_raw + 2 * (Sh::QBytes + 32 + Sh::MergeBytes)) + warp * 64;
                __syncwarp();
                if (!(t & 1)) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        wx[32 * col + 16 * x + g] = digit_bits_pos(e[x].x, f);
                        wx[32 * col + 16 * x + 8 + g] = digit_bits_pos(e[x].y, f);
                    }
                }
                __syncwarp();
                const int dig = g & 3;
                const uint32_t sel = (uint32_t)dig | ((uint32_t)(4 + dig) << 4), flip = dig < 2 ? 0x80808080u : 0u, keep = dig < 3 ? ~0u : 0u;
                uint32_t wb[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint4 y = *reinterpret_cast<const uint4*>(wx + 32 * (g >> 2) + 16 * b + 4 * t);
                    wb[b] = (__byte_perm(__byte_perm(y.x, y.y, sel), __byte_perm(y.z, y.w, sel), 0x5410) ^ flip) & keep;
                }
                // output: row g of tile x is element (DP/8) g + 2 x, row g + 8 the next: four keys'
                // bytes of one element make one A register
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
                        int c[4];
                        mma_s8_first(c, a[0][2 * k], a[0][2 * k + 1], a[1][2 * k], a[1][2 * k + 1], wb[0], wb[1]);
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            o[4 * w + 2 * k + r] = fma2(pack2((float)c[2 * r], (float)c[2 * r + 1]), pack2(u, u),
                                                        mul2(o[4 * w + 2 * k + r], pack2(back, back)));
                    }
                }
            } else {
                uint32_t wd[2][3];                                             // digits of a block's four weights
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    digits4(digit_bits_pos(e[2 * b].x, f), digit_bits_pos(e[2 * b].y, f), digit_bits_pos(e[2 * b + 1].x, f),
                            digit_bits_pos(e[2 * b + 1].y, f), wd[b]);
                // output: column n of tile x is element (DP/8) n + x: four keys' bytes of one
                // element make one B register
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
                    int hi[4][4], lo[4][4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_s8_first(hi[k], wd[0][2], wd[0][1], wd[1][2], wd[1][1], a[0][k], a[1][k]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_s8_first(lo[k], wd[0][0], wd[0][0], wd[1][0], wd[1][0], a[0][k], a[1][k]);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        o[4 * w + k] = fma2(join_digits(hi[k][0], hi[k][1], hi[k][2], hi[k][3], lo[k][0], lo[k][1]), pack2(u, u),
                                            mul2(o[4 * w + k], pack2(back, back)));
                }
            }
            load_values(na0, na1);
            a0 = na0; a1 = na1;
            j += kSplitWarps * 32;
        } while (j < cur.jend);
        // this warp's columns: sum over the lanes of a column, then all to shared memory
        float* mo = reinterpret_cast<float*>(ps_raw + 2 * (Sh::QBytes + 32) + buf * Sh::MergeBytes);   // [4][8][DP + 4]
        float l = unpack2(l2).x + unpack2(l2).y;
        float* ow = mo + (warp * NC + col) * (DP + 4);
        if constexpr (kNarrow) {
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            float v[Sh::NT];                                               // the digits together
#pragma unroll
            for (int x = 0; x < Sh::NT; ++x) {
                const float2 c = unpack2(o[x]);
                v[x] = t & 1 ? c.x * 65536.0f : ffma(c.y, 256.0f, c.x);
                v[x] += __shfl_xor_sync(0xffffffffu, v[x], 1);
            }
            if (!(t & 1) && col < cur.cols) {
                if (g == 0) { ow[DP] = m; ow[DP + 1] = l; }
#pragma unroll
                for (int x = 0; x < Sh::NT; x += 4)
                    *reinterpret_cast<float4*>(ow + (DP / 8) * g + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
            }
        } else if (l += __shfl_xor_sync(0xffffffffu, l, 1), l += __shfl_xor_sync(0xffffffffu, l, 2); col < cur.cols) {
            if (t == 0) { ow[DP] = m; ow[DP + 1] = l; }
#pragma unroll
            for (int x = 0; x < Sh::NT; x += 4) {
                const float2 a = unpack2(o[x]), b = unpack2(o[x + 1]), c = unpack2(o[x + 2]), d = unpack2(o[x + 3]);
                *reinterpret_cast<float4*>(ow + (DP / 4) * t + x) = make_float4(a.x, b.x, c.x, d.x);
                *reinterpret_cast<float4*>(ow + (DP / 4) * t + DP / 8 + x) = make_float4(a.y, b.y, c.y, d.y);
            }
        }
        if (!kNarrow && nxt.it.s >= 0) put_queries(nxt, buf ^ 1);
        __syncthreads();
        // (narrow: not by the warp that also has the next queries to fetch)
        for (int i = tid; i < cur.cols * (DP / 4); i += kSplitWarps * 32) {
            const int col = i / (DP / 4), d = 4 * (i % (DP / 4)), cc = cur.col0 + col, tok = cur.it.len == 1 ? 0 : cc / p.G;
            const int splits = row_splits(p, pos0 + tok);
            if (d >= dh || cur.it.split >= splits) continue;
            const float* mc = mo + col * (DP + 4);
            constexpr int W = NC * (DP + 4);
            float M = -INFINITY, L = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kSplitWarps; ++w) M = fmaxf(M, mc[w * W + DP]);
            const float B = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < kSplitWarps; ++w) {
                const float e = exp2_fast(mc[w * W + DP] - B);
                const float4 x = *reinterpret_cast<const float4*>(mc + w * W + d);
                L = ffma(mc[w * W + DP + 1], e, L);
                acc.x = ffma(x.x, e, acc.x); acc.y = ffma(x.y, e, acc.y);
                acc.z = ffma(x.z, e, acc.z); acc.w = ffma(x.w, e, acc.w);
            }
            const int row = cur.it.a + tok, h = cur.kvh() * p.G + cc - tok * p.G;
            if (splits == 1) {
                const float inv = L == 0.0f ? 0.0f : fdiv(1.0f, L);
                *reinterpret_cast<float4*>(p.out + (size_t)row * p.ldo + (size_t)h * dh + d) =
                    make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                float* pp = few_part(p, cur.seq(), tok, row, h, cur.it.split);
                *reinterpret_cast<float4*>(pp + d) = acc;
                if (d == 0) { pp[dh] = M; pp[dh + 1] = L; }
            }
        }
        if (nxt.it.s < 0) return;
        cur = nxt;
    }
}

// ---- many rows per sequence, d_head above 128 (three digits' output sums of 256 elements do
// not fit the tensor memory beside anything): a CTA of 4 warps takes 64 rows ((token, head) pairs of
// one KV head), warp w 16 of them, against a split of the keys in tiles of KT. A =
// query or weight digits (rows x 32), B = codes: keys as they lie, values turned to
// [d][key] on their way into shared memory (byte permutes, once for the CTA). The
// key order inside a B fragment of the values is the one that the score fragments
// already have, so weights go from scores to A fragments inside their thread.
// Codes of tile i + 1 are on their way while tile i is computed.
constexpr int kTileRows = 64;

struct TileShape {
    static constexpr int DP = 256;                             // d_head, padded
    static constexpr int KT = 64;                              // keys per tile
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

static __global__ void __launch_bounds__(128, 1) paged_attn_tile_kernel(const __grid_constant__ PagedAttnParams p) {
    using Sh = TileShape;
    constexpr int DP = Sh::DP, KT = Sh::KT, NB = Sh::NB;
    extern __shared__ __align__(16) unsigned char pt_raw[];
    uint8_t* qd = pt_raw;                                      // A fragments [3][4 warps][DP / 32][lane][16]
    uint8_t* kt = qd + Sh::QBytes;                             // [2][KT][DP]
    uint8_t* vt = kt + 2 * Sh::KBytes;                         // [2][DP][KT]
    float* sq = reinterpret_cast<float*>(vt + 2 * Sh::KBytes); // [64]
    float* sc = sq + kTileRows;                                // [2][3][NB]: key scales, value scales, 1 where there
    long long* cell = reinterpret_cast<long long*>(sc + 6 * NB);   // [2][NB] a tile's blocks in the pool
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int dh = p.c.dh, psz = 1 << p.c.page_log2;

    after_previous();
    const AttnItem it = find_item<kTileRows>(p, blockIdx.x, lane);
    if (it.s < 0) return;
    const int row0 = it.tile * kTileRows, rows = min(it.len * p.G - row0, kTileRows);
    const int pos0 = it.kv - it.len;
    const int n = min(pos0 + (row0 + rows - 1) / p.G + 1, p.r.cap);      // keys that any row sees
    const int j0 = it.split << p.kc_log2, jend = min(n, j0 + (1 << p.kc_log2));
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
            sc[3 * NB * b + tid] = cb >= 0 ? (tid < NB ? p.c.ks : p.c.vs)[cb] : 0.0f;
            if (tid < NB) sc[3 * NB * b + 2 * NB + tid] = cb >= 0 ? 1.0f : 0.0f;
            if (cb == -1) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
        }
    };
    // This thread's part of a value tile: in block vb four keys vq2 + {0, 1, 8, 9} of two
    // 16-element columns from d0.
    constexpr int VC = KT * DP / 64 / 128;                     // 16-byte columns a thread turns
    const int vb = (lane & 15) >> 2, vq2 = (lane & 3) * 2, d0 = 16 * VC * (2 * warp + (lane >> 4));
    uint4 vr[VC][4];
    auto load_values = [&](int i) {
        const long long at = cell[NB * (i & 1) + vb];
#pragma unroll
        for (int x = 0; x < VC; ++x) {
            // what is not there is read from the pool's first block: its weights are 0, and
            // elements past dh are not stored
            const int d = d0 + 16 * x < dh ? d0 + 16 * x : 0;
            const int8_t* src = p.c.v + (max(at, 0ll) * kKvBlock + vq2) * dh + d;
#pragma unroll
            for (int k = 0; k < 4; ++k) vr[x][k] = *reinterpret_cast<const uint4*>(src + ((k >> 1) * 8 + (k & 1)) * dh);
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
                    *reinterpret_cast<uint32_t*>(vd + unit_at<KT>(d0 + 16 * x + 4 * w + z, vq2 >> 1) + 4 * vb) = y[z];
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
            const float f0 = weight_factor(wt0), f1 = weight_factor(wt1);
            u0 = wt0 < INFINITY ? weight_unit(f0) : __int_as_float(0x7fffffff);
            u1 = wt1 < INFINITY ? weight_unit(f1) : __int_as_float(0x7fffffff);
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
                uint4 b[2];
#pragma unroll
                for (int z = 0; z < 2; ++z) b[z] = *reinterpret_cast<const uint4*>(vd + unit_at<KT>(8 * (x + z) + g, t));
#pragma unroll
                for (int e = 0; e < 3; ++e)
#pragma unroll
                    for (int z = 0; z < 2; ++z) mma_s8_first(c[z][e], wa[0][e][0], wa[0][e][1], wa[0][e][2], wa[0][e][3], b[z].x, b[z].y);
#pragma unroll
                for (int e = 0; e < 3; ++e)
#pragma unroll
                    for (int z = 0; z < 2; ++z) mma_s8(c[z][e], wa[1][e][0], wa[1][e][1], wa[1][e][2], wa[1][e][3], b[z].z, b[z].w);
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
        float* dst = splits > 1 ? many_part(p, row, h, it.split)
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

// ---- many rows per sequence, d_head up to 128: the 5th-generation tensor cores. A CTA
// takes 128 rows against a split of the keys in tiles of 128.
//   S = Q K^T, O = W V, each three MMA chains (tcgen05 kind::i8, one per digit) of
//   128 x 128 x d_head (x 128 keys). The passes S(0) S(1) O(0) S(2) O(1) ... take their
//   three blocks of 128 TMEM columns from a ring of four: a pass's first chain needs the
//   pass before the last one read, its others the last one. So MMAs run while the
//   softmax warps work on what they have read before; what bounds the kernel is the
//   latency of that work, since all four of a row's warps meet every tile: scores 1000
//   clocks, exponentials 1800, digits 1700, folding 1200 of about 7500 a tile (traced with
//   a ring of three blocks). 4 x 2047 rows, 32 / 8 heads of 128: 598 us, 54 % of the issue
//   slots, tensor pipe active 16 %.
// Warps 0 .. 15, softmax: warp w reads TMEM lanes 32 (w % 4) .. + 31, a row a thread, and
//   set w / 4 has keys 32 (w / 4) .. + 31 of the tile and elements 32 (w / 4) .. + 31 of the
//   output: no shuffles; a row's four threads exchange (maximum, largest weight) through
//   shared memory, a barrier of 128 threads.
// Warps 16 .. 18, copies: keys by cp.async, values turned to [element][key] by byte
//   permutes, both in the 128-byte-swizzled K-major layout, two buffers each; scales.
// Warp 19: issues the MMAs. (20 warps: 96 registers a thread; 21 would leave 80.)
// Every wait is bounded; a warp whose wait ran out goes on without waiting (its barriers
// still meet), sets the error word and the outputs are garbage.
constexpr int kMmaRows = 128;
constexpr int kMmaKeys = 128;
constexpr int kMmaSoftWarps = 16;
constexpr int kMmaCopyWarps = 3;
constexpr int kMmaThreads = (kMmaSoftWarps + kMmaCopyWarps + 1) * 32;

struct MmaSmem {
    static constexpr int Tile = 128 * 128;                     // one 128 x 128-byte operand
    static constexpr int Q = 0;                                // [3 digits]
    static constexpr int P = Q + 3 * Tile;                     // [2 tiles][3 digits] weights
    static constexpr int K = P + 6 * Tile;                     // [2]
    static constexpr int V = K + 2 * Tile;                     // [2]
    static constexpr int Xm = V + 2 * Tile;                    // [2][4 sets][128 rows] (maximum, largest weight)
    static constexpr int Sc = Xm + 2 * 4 * 128 * 8;            // [4 tiles][3][8]: key scales, value scales, 1 where there
    static constexpr int Sq = Sc + 4 * 24 * 4;                 // [128] units of the rows' scores
    static constexpr int Bars = Sq + 128 * 4;                  // 16 barriers, TMEM address, fail
    static constexpr int Bytes = Bars + 16 * 8 + 16;
    static constexpr int OutStride = 132;                      // floats a row of the staged output (in P)
    static constexpr int Alloc = Bytes + 1024;                 // operands start on 1024 bytes
};

static __global__ void __launch_bounds__(kMmaThreads, 1) paged_attn_mma_kernel(const __grid_constant__ PagedAttnParams p) {
    using Sm = MmaSmem;
    extern __shared__ unsigned char pm_raw[];
    unsigned char* sm = pm_raw + ((1024u - (smem_u32(pm_raw) & 1023u)) & 1023u);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + Sm::Bars);      // [2] copies -> MMA
    uint64_t* kempty = kfull + 2;                                      // [2] MMA -> copies
    uint64_t* vfull = kempty + 2;                                      // [2]
    uint64_t* vempty = vfull + 2;                                      // [2]
    uint64_t* sfull = vempty + 2;                                      // scores in TMEM
    uint64_t* sfree = sfull + 1;                                       // scores read
    uint64_t* pfull = sfree + 1;                                       // [2] weights written
    uint64_t* ofull = pfull + 2;                                       // output sums in TMEM
    uint64_t* ofree = ofull + 1;                                       // output sums read
    uint64_t* done = ofree + 1;                                        // every MMA complete
    uint64_t* qfull = done + 1;                                        // query digits written
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float2* xm = reinterpret_cast<float2*>(sm + Sm::Xm);
    float* sc = reinterpret_cast<float*>(sm + Sm::Sc);
    float* sq = reinterpret_cast<float*>(sm + Sm::Sq);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int dh = p.c.dh, psz = 1 << p.c.page_log2;

    after_previous();
    const AttnItem it = find_item<kMmaRows>(p, blockIdx.x, lane);
    if (it.s < 0) return;
    const int row0 = it.tile * kMmaRows, rows = min(it.len * p.G - row0, kMmaRows);
    const int pos0 = it.kv - it.len;
    const int n = min(pos0 + (row0 + rows - 1) / p.G + 1, p.r.cap);      // keys that any row sees
    const int j0 = it.split << p.kc_log2, jend = min(n, j0 + (1 << p.kc_log2));
    if (j0 >= n && it.split > 0) return;
    const int ntiles = max((jend - j0 + kMmaKeys - 1) / kMmaKeys, 0);

    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(&kfull[b], kMmaCopyWarps * 32); mbar_init(&kempty[b], 1);
            mbar_init(&vfull[b], kMmaCopyWarps * 32); mbar_init(&vempty[b], 1);
            mbar_init(&pfull[b], kMmaSoftWarps);
        }
        mbar_init(sfull, 2); mbar_init(sfree, kMmaSoftWarps);
        mbar_init(ofull, 1); mbar_init(ofree, kMmaSoftWarps); mbar_init(done, 1); mbar_init(qfull, kMmaSoftWarps);
        fence_mbar_init();
        *fail = 0;
    }
    if (warp == kMmaSoftWarps + kMmaCopyWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool dead = false;                                         // a wait ran out: wait no more
    // bounded (1 s); `pause` ns between polls, which take issue slots from the warps that work
    auto wait = [&](uint64_t* bar, int parity, unsigned pause) {
        if (dead || mbar_try_wait(bar, (uint32_t)parity)) return;
        const uint64_t t0 = globaltimer_ns();
        for (unsigned k = 1; !mbar_try_wait(bar, (uint32_t)parity); ++k) {
            __nanosleep(pause);
            if ((k & 63u) == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
                dead = true;
                *fail = 1;
                return;
            }
        }
    };
    auto wait_warp = [&](uint64_t* bar, int parity, unsigned pause) {   // by a whole warp
        wait(bar, parity, pause);
        dead = __any_sync(0xffffffffu, dead);
    };

    if (warp == kMmaSoftWarps + kMmaCopyWarps) {
        // ---- MMAs (one lane)
        if (lane == 0) {
            const uint32_t id = umma_idesc_i8(128, true), base = smem_u32(sm);
            const int ksteps = (dh + 31) / 32;
            // chain e (digit 2 - e) of pass `op`: operands at a + (2 - e) tiles and b, `steps` of 32 bytes
            auto chain = [&](int op, int e, uint32_t a, uint32_t b, int steps) {
                const uint32_t col = 128u * ((3 * op + e) & 3);
                for (int k = 0; k < steps; ++k)
                    umma_i8(tmem + col, umma_desc_sw128(a + (2 - e) * Sm::Tile + 32 * k), umma_desc_sw128(b + 32 * k), id, k > 0 ? 1u : 0u);
            };
            // S(i): pass 2 i - 1 (0: pass 0), after O(i - 2) (pass 2 i - 2) and S(i - 1) (2 i - 3)
            auto scores = [&](int i) {
                const int op = max(2 * i - 1, 0);
                const uint32_t kb = base + Sm::K + (i & 1) * Sm::Tile;
                wait(&kfull[i & 1], (i >> 1) & 1, 20);
                if (i == 1) wait(sfree, 0, 20);                // (later ones: waited for by O(i - 2))
                tc_fence_after();
                chain(op, 0, base + Sm::Q, kb, ksteps);
                if (i > 1) {
                    wait(ofree, i & 1, 20);
                    tc_fence_after();
                }
                chain(op, 1, base + Sm::Q, kb, ksteps);
                chain(op, 2, base + Sm::Q, kb, ksteps);
                umma_commit(&kempty[i & 1]);
                umma_commit(sfull);
                mbar_arrive(sfull);                            // passes on what the copies wrote: the scales
            };
            // O(i): pass 2 i + 2, after S(i + 1) (2 i + 1) and O(i - 1) (2 i, whose reading the pass
            // before has waited for, except at the end, where there is no S(i + 1))
            auto output = [&](int i) {
                const uint32_t pb = base + Sm::P + 3 * (i & 1) * Sm::Tile, vb = base + Sm::V + (i & 1) * Sm::Tile;
                const bool end = i == ntiles - 1;
                if (end && i > 0) wait(ofree, (i - 1) & 1, 20);
                if (end && i == 0) wait(sfree, 0, 20);         // (no S(1) has waited for S(0))
                wait(&pfull[i & 1], (i >> 1) & 1, 20);
                wait(&vfull[i & 1], (i >> 1) & 1, 20);
                tc_fence_after();
                chain(2 * i + 2, 0, pb, vb, kMmaKeys / 32);
                if (!end) {
                    wait(sfree, (i + 1) & 1, 20);
                    tc_fence_after();
                }
                chain(2 * i + 2, 1, pb, vb, kMmaKeys / 32);
                chain(2 * i + 2, 2, pb, vb, kMmaKeys / 32);
                umma_commit(&vempty[i & 1]);
                umma_commit(ofull);
            };
            if (ntiles > 0) {
                wait(qfull, 0, 20);
                scores(0);
            }
            for (int i = 0; i < ntiles; ++i) {
                if (i > 0) output(i - 1);
                if (i + 1 < ntiles) scores(i + 1);
            }
            if (ntiles > 0) output(ntiles - 1);
            umma_commit(done);                                 // also after a wait that ran out: no MMA may
            if (!mbar_wait_bounded(done, 0)) *fail = 1;        // be under way when its memory is given up
        }
    } else if (warp >= kMmaSoftWarps) {
        // ---- copies
        const int ct = tid - kMmaSoftWarps * 32, cw = warp - kMmaSoftWarps;
        for (int i = 0; i < ntiles; ++i) {
            const int j = j0 + i * kMmaKeys, b = i & 1;
            // the tile's blocks in the pool, block `lane & 7` (-1: page outside it, -2: past the end)
            long long cell = -2;
            const int jb = j + 16 * (lane & 7);
            if (jb < jend) {
                const int page = page_of(p.c, p.r, it.s, jb);
                cell = page < 0 ? -1 : ((long long)page * p.c.KVH + it.kvh) * (psz >> 4) + ((jb & (psz - 1)) >> 4);
            }
            if (i > 1) wait_warp(&kempty[b], ((i >> 1) - 1) & 1, 200);
            unsigned char* kd = sm + Sm::K + b * Sm::Tile;
            auto cell_of = [&](int blk) {                      // (whole warps)
                return (long long)(((unsigned long long)(unsigned)__shfl_sync(0xffffffffu, (int)(cell >> 32), blk) << 32) |
                                   (unsigned)__shfl_sync(0xffffffffu, (int)cell, blk));
            };
#pragma unroll
            for (int x = 0; x < (1024 + kMmaCopyWarps * 32 - 1) / (kMmaCopyWarps * 32); ++x) {
                const int unit = x * kMmaCopyWarps * 32 + ct, u = unit & 7, key = unit >> 3;
                if (unit >= 1024) break;                       // (whole warps)
                const long long at = cell_of(key >> 4);
                const bool there = at >= 0 && 16 * u < dh;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                             ::"r"(smem_u32(kd + key * 128 + ((u ^ (key & 7)) << 4))),
                               "l"(p.c.k + (there ? (at * kKvBlock + (key & 15)) * dh + 16 * u : 0)), "r"(there ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            // values: keys 4 lane .. + 3 of 16-element columns cw, cw + 3, cw + 6
            uint4 vr[3][4];
            {
                const long long at = max(cell_of(lane >> 2), 0ll);     // what is not there has no weight
                const int8_t* src = p.c.v + (at * kKvBlock + 4 * (lane & 3)) * dh;
#pragma unroll
                for (int x = 0; x < 3; ++x) {
                    const int d = 16 * (cw + 3 * x) < dh ? 16 * (cw + 3 * x) : 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) vr[x][k] = *reinterpret_cast<const uint4*>(src + k * dh + d);
                }
            }
            if (ct < 8) {
                float* s = sc + (i & 3) * 24 + ct;
                s[0] = cell >= 0 ? p.c.ks[cell] : 0.0f;
                s[8] = cell >= 0 ? p.c.vs[cell] : 0.0f;
                s[16] = cell >= 0 ? 1.0f : 0.0f;
                if (cell == -1) set_err(p.err, B2_DEV_ERR_BAD_PAGE);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            fence_async_smem();
            mbar_arrive(&kfull[b]);
            if (i > 1) wait_warp(&vempty[b], ((i >> 1) - 1) & 1, 200);
            unsigned char* vd = sm + Sm::V + b * Sm::Tile;
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                if (cw + 3 * x >= 8) break;
                const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vr[x][0]);
                const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vr[x][1]);
                const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vr[x][2]);
                const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vr[x][3]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t a = __byte_perm(w0[w], w1[w], 0x5140), c = __byte_perm(w2[w], w3[w], 0x5140);
                    const uint32_t d = __byte_perm(w0[w], w1[w], 0x7362), e = __byte_perm(w2[w], w3[w], 0x7362);
                    const uint32_t y[4] = {__byte_perm(a, c, 0x5410), __byte_perm(a, c, 0x7632), __byte_perm(d, e, 0x5410),
                                           __byte_perm(d, e, 0x7632)};
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int el = 16 * (cw + 3 * x) + 4 * w + z;
                        *reinterpret_cast<uint32_t*>(vd + el * 128 + (((lane >> 2) ^ (el & 7)) << 4) + 4 * (lane & 3)) = y[z];
                    }
                }
            }
            fence_async_smem();
            mbar_arrive(&vfull[b]);
        }
    } else {
        // ---- softmax and output
        // queries -> digits: 16 lanes a row (rows past the last are zeros)
#pragma unroll
        for (int x = 0; x < kMmaRows / 32; ++x) {
            const int l16 = tid & 15, r = 32 * x + (tid >> 4), cc = row0 + r;
            const float* qr = p.q + (size_t)(it.a + cc / p.G) * p.ldq + (size_t)(it.kvh * p.G + cc % p.G) * dh;
            query_digits<128>(qr, r < rows, dh, l16, [&](int e, int d, uint32_t w) {
                *reinterpret_cast<uint32_t*>(sm + Sm::Q + e * Sm::Tile + r * 128 + (((d >> 4) ^ (r & 7)) << 4) + (d & 15)) = w;
            }, sq + r);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);
        asm volatile("bar.sync 5, 512;" ::: "memory");         // the units, too
        const int quarter = warp & 3, set = warp >> 2, row = 32 * quarter + lane, col0 = 32 * set;
        const uint32_t trow = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)col0;
        const int lim = row < rows ? min(pos0 + (row0 + row) / p.G + 1, n) : 0;   // keys the row sees
        const int wmin = __reduce_min_sync(0xffffffffu, lim), wmax = __reduce_max_sync(0xffffffffu, lim);
        const float sqr = sq[row];
        float m = -INFINITY, l = 0.0f;                         // l: this set's keys
        float back = 1.0f, u = 0.0f;                           // of the tile whose output is pending
        bool pending = false;                                  // that output has this row quarter's weights
        f32x2 o[16];                                           // elements col0 + 2 x, + 1
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] = 0ull;
        // 8 columns from col0 + 8 q of a pass's digit e (chain 2 - e)
        auto read8 = [&](int op, int e, int q, uint32_t (&c)[8]) { tmem_ld8(trow + 128u * ((3 * op + 2 - e) & 3) + 8u * q, c); };
        auto fold = [&](int i) {                               // output sums of tile i
            wait_warp(ofull, i & 1, 20);
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (!pending || col0 + 8 * q >= dh) continue;  // (the same for the whole warp)
                uint32_t c[3][8];
#pragma unroll
                for (int e = 0; e < 3; ++e) read8(2 * i + 2, e, q, c[e]);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    o[4 * q + x] = fma2(join_digits((int)c[2][2 * x], (int)c[2][2 * x + 1], (int)c[1][2 * x], (int)c[1][2 * x + 1],
                                                    (int)c[0][2 * x], (int)c[0][2 * x + 1]),
                                        pack2(u, u), mul2(o[4 * q + x], pack2(back, back)));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ofree);
        };
        for (int i = 0; i < ntiles; ++i) {
            const int j = j0 + i * kMmaKeys;
            const bool busy = wmax > j;                        // the same for the quarter's four warps
            wait_warp(sfull, i & 1, 20);
            tc_fence_after();
            float2 s[16];                                      // keys j + col0 + 2 x, + 1
            const float* scb = sc + (i & 3) * 24 + 2 * set;
            if (busy) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t c[3][8];
#pragma unroll
                    for (int e = 0; e < 3; ++e) read8(max(2 * i - 1, 0), e, q, c[e]);
                    tmem_wait_ld();
                    const float us = sqr * scb[q >> 1];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        s[4 * q + x] = unpack2(mul2(join_digits((int)c[2][2 * x], (int)c[2][2 * x + 1], (int)c[1][2 * x], (int)c[1][2 * x + 1],
                                                                (int)c[0][2 * x], (int)c[0][2 * x + 1]), pack2(us, us)));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sfree);
            float nback = 1.0f, nu = 0.0f;
            if (busy) {
                const float t0 = scb[16], t1 = scb[17], v0 = scb[8], v1 = scb[9];
                const int jk = j + col0;
                if (jk + 32 > wmin || t0 + t1 != 2.0f) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int lx = (x < 8 ? t0 : t1) != 0.0f ? lim : 0;
                        if (jk + 2 * x >= lx) s[x].x = -INFINITY;
                        if (jk + 2 * x + 1 >= lx) s[x].y = -INFINITY;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 16; ++x) mx = fmaxf(mx, fmaxf(s[x].x, s[x].y));
                // exponentials and weights p v_scale relative to the set's own maximum. A score that
                // is not a number makes l NaN, which is enough; a value scale that is not one
                // needs checks
                const float h = mx == -INFINITY ? 0.0f : mx;
                f32x2 ls = 0ull;
                float wt = 0.0f;
                const bool sane = v0 + v1 == v0 + v1;
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float2 z = unpack2(add2(pack2(s[x].x, s[x].y), pack2(-h, -h)));
                    const f32x2 ev = pack2(exp2_fast(z.x), exp2_fast(z.y));
                    ls = add2(ls, ev);
                    const float v = x < 8 ? v0 : v1;
                    s[x] = unpack2(mul2(ev, pack2(v, v)));
                }
                if (!sane) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {             // a masked key weighs nothing, whatever its scale
                        if (jk + 2 * x >= lim) s[x].x = 0.0f;
                        if (jk + 2 * x + 1 >= lim) s[x].y = 0.0f;
                        if (s[x].x != s[x].x || s[x].y != s[x].y) wt = INFINITY;
                    }
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) wt = fmaxf(wt, fmaxf(s[x].x, s[x].y));
                // the other sets' keys: common maximum, one factor for all weights
                float2* xt = xm + (i & 1) * 512 + row;
                xt[128 * set] = make_float2(mx, wt);
                asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
                float2 y[4];
                float top = m;
#pragma unroll
                for (int q = 0; q < 4; ++q) { y[q] = xt[128 * q]; top = fmaxf(top, y[q].x); }
                const float b = top == -INFINITY ? 0.0f : top;
                nback = exp2_fast(m - b);
                m = top;
                const float corr = exp2_fast(mx - b);
                l = ffma(l, nback, (unpack2(ls).x + unpack2(ls).y) * corr);
                float big = 0.0f;
                bool nan = false;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    big = fmaxf(big, y[q].y * exp2_fast(y[q].x - b));
                    nan |= y[q].y == INFINITY;
                }
                const float f = weight_factor(big), fe = f * corr;
                nu = nan ? __int_as_float(0x7fffffff) : weight_unit(f);
                unsigned char* pd = sm + Sm::P + 3 * (i & 1) * Sm::Tile + row * 128;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {               // 16 keys: one 16-byte unit a digit
                    uint32_t w[3][4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float2 a = s[8 * hh + 2 * x], c = s[8 * hh + 2 * x + 1];
                        const float2 z0 = unpack2(fma2(pack2(a.x, a.y), pack2(fe, fe), pack2(kDigitBase, kDigitBase)));
                        const float2 z1 = unpack2(fma2(pack2(c.x, c.y), pack2(fe, fe), pack2(kDigitBase, kDigitBase)));
                        uint32_t d[3];
                        digits4(__float_as_uint(z0.x), __float_as_uint(z0.y), __float_as_uint(z1.x), __float_as_uint(z1.y), d);
                        w[0][x] = d[0]; w[1][x] = d[1]; w[2][x] = d[2];
                    }
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        *reinterpret_cast<uint4*>(pd + e * Sm::Tile + (((2 * set + hh) ^ (row & 7)) << 4)) =
                            make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
                }
                fence_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[i & 1]);
            if (i > 0) fold(i - 1);
            back = nback; u = nu; pending = busy;
        }
        if (ntiles > 0) fold(ntiles - 1);
        // the row's sum over its four sets
        xm[set * 128 + row].x = l;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
        float L = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) L += xm[q * 128 + row].x;
        // the rows through shared memory (the weights are not needed any more), so that a warp
        // writes one row at a time
        float* so = reinterpret_cast<float*>(sm + Sm::P);
        const int splits = row < rows ? row_splits(p, pos0 + (row0 + row) / p.G) : 1;
        const float inv = splits > 1 ? 1.0f : L == 0.0f ? 0.0f : fdiv(1.0f, L);
#pragma unroll
        for (int x = 0; x < 16; x += 2) {
            const float2 a = unpack2(o[x]), c = unpack2(o[x + 1]);
            *reinterpret_cast<float4*>(so + row * Sm::OutStride + col0 + 2 * x) = make_float4(a.x * inv, a.y * inv, c.x * inv, c.y * inv);
        }
        if (set == 0) xm[512 + row] = make_float2(m, L);
        asm volatile("bar.sync 5, 512;" ::: "memory");
        for (int r = warp; r < rows; r += kMmaSoftWarps) {
            const int cc = row0 + r, tok = cc / p.G, ns = row_splits(p, pos0 + tok);
            const int orow = it.a + tok, h = it.kvh * p.G + cc - tok * p.G;
            if (it.split >= ns) continue;
            float* dst = ns > 1 ? many_part(p, orow, h, it.split)
                                : p.out + (size_t)orow * p.ldo + (size_t)h * dh;
            if (4 * lane < dh) *reinterpret_cast<float4*>(dst + 4 * lane) = *reinterpret_cast<const float4*>(so + r * Sm::OutStride + 4 * lane);
            if (ns > 1 && lane < 2) dst[dh + lane] = lane ? xm[512 + r].y : xm[512 + r].x;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaSoftWarps + kMmaCopyWarps) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (tid == 0 && *fail) set_err(p.err, B2_DEV_ERR_TIMEOUT);
}

// Joins a (row, head)'s splits in a fixed order: WPH warps a pair, warp w the splits w,
// w + WPH, ..., then the warps in order. Bound by latency: the splits' maxima and sums are
// read a lane each, so that the partial outputs' loads depend on nothing and overlap.
// (One warp for 79 splits took 35 us where the attention itself took 26.) Grid (rows,
// heads * WPH / 8).
template <int WPH>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const __grid_constant__ PagedAttnParams p) {
    __shared__ __align__(16) float so[8][256];
    __shared__ float sm[8][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dh = p.c.dh;
    const int h = blockIdx.y * (8 / WPH) + warp / WPH, part = warp % WPH;
    after_previous();                                              // the splits are written
    int n = 0, row = blockIdx.x, s = 0, tok = 0;                   // the row's splits, the same for the whole CTA
    bool few = true;
    if (p.join_rows) {
        s = blockIdx.x / p.join_rows;
        tok = blockIdx.x % p.join_rows;
        const SeqRows q = seq_rows(p.r, s);
        row = q.a + tok;
        if (tok < q.len && (long long)q.len * p.G <= p.few) n = splits_of(p.kc_few, min(q.pos0() + tok + 1, p.r.cap));
    } else {
        for (int base = 0; base < p.r.n_seq && n == 0; base += 32) {
            SeqRows q{0, 0, 0};
            if (base + lane < p.r.n_seq) q = seq_rows(p.r, base + lane);
            const unsigned m = __ballot_sync(0xffffffffu, row >= q.a && row < q.a + q.len);
            if (m) {
                const int src = __ffs(m) - 1, pos = __shfl_sync(0xffffffffu, q.pos0() + row - q.a, src);
                s = base + src;
                tok = row - __shfl_sync(0xffffffffu, q.a, src);
                few = (long long)__shfl_sync(0xffffffffu, q.len, src) * p.G <= p.few;
                n = splits_of(few ? p.kc_few : p.kc_many, min(pos + 1, p.r.cap));
            }
        }
    }
    if (n < 2) return;
    const int stride = dh + 4, hc = min(h, p.H - 1);
    const float* base = few ? few_part(p, s, tok, row, hc, 0) : many_part(p, row, hc, 0);
    float M = -INFINITY, L = 0.0f;
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int s0 = part; s0 < n; s0 += 32 * WPH) {                  // 32 of this warp's splits at a time
        const int s = s0 + lane * WPH;
        const bool live = s < n;
        const float ms = live ? base[(size_t)s * stride + dh] : -INFINITY, ls = live ? base[(size_t)s * stride + dh + 1] : 0.0f;
        float top = ms;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, M);
        const float B = top == -INFINITY ? 0.0f : top, back = exp2_fast(M - B), e = live ? exp2_fast(ms - B) : 0.0f;
        M = top;
        float add = e * ls;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) add += __shfl_xor_sync(0xffffffffu, add, x);
        L = ffma(L, back, add);
#pragma unroll
        for (int i = 0; i < 2; ++i) { acc[i].x *= back; acc[i].y *= back; acc[i].z *= back; acc[i].w *= back; }
        const int cnt = min((n - s0 + WPH - 1) / WPH, 32);
#pragma unroll 8
        for (int k = 0; k < cnt; ++k) {
            const float w = __shfl_sync(0xffffffffu, e, k);
            const float* ps = base + (size_t)(s0 + k * WPH) * stride;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 4 * lane + 128 * i;
                if (d >= dh) continue;
                const float4 x = *reinterpret_cast<const float4*>(ps + d);
                acc[i].x = ffma(x.x, w, acc[i].x); acc[i].y = ffma(x.y, w, acc[i].y);
                acc[i].z = ffma(x.z, w, acc[i].z); acc[i].w = ffma(x.w, w, acc[i].w);
            }
        }
    }
    if constexpr (WPH > 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (4 * lane + 128 * i < dh) *reinterpret_cast<float4*>(&so[warp][4 * lane + 128 * i]) = acc[i];
        if (lane == 0) { sm[warp][0] = M; sm[warp][1] = L; }
        __syncthreads();
        if (part != 0) return;
        M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WPH; ++w) M = fmaxf(M, sm[warp + w][0]);
        const float B = M == -INFINITY ? 0.0f : M;
        L = 0.0f;
        acc[0] = acc[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WPH; ++w) {
            const float e = exp2_fast(sm[warp + w][0] - B);
            L = ffma(sm[warp + w][1], e, L);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (4 * lane + 128 * i >= dh) continue;
                const float4 x = *reinterpret_cast<const float4*>(&so[warp + w][4 * lane + 128 * i]);
                acc[i].x = ffma(x.x, e, acc[i].x); acc[i].y = ffma(x.y, e, acc[i].y);
                acc[i].z = ffma(x.z, e, acc[i].z); acc[i].w = ffma(x.w, e, acc[i].w);
            }
        }
    }
    if (h >= p.H) return;
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
