// paged_rows.cuh — what the kernels over the paged 8-bit KV cache share (paged.cuh,
// tree.cuh): the cache and the rows of a call as kernels see them, loads behind the
// launch before, packed f32 arithmetic.
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

// which of n_src rows an index picks for row `row` of a call (-1: none)
__device__ __forceinline__ int picked_row(const int* index, int row, int n_src, int* err) {
    const int at = index[row];
    if ((unsigned)at < (unsigned)n_src) return at;
    set_err(err, B2_DEV_ERR_BAD_ROW);
    return -1;
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

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Joins the n partial results [dh + 4] (o, m in base 2, l) at `base` of one (row, head) into `out`
// (nullptr: the warp has none and only meets the others): by WPH warps of a CTA of 8, this
// one number `part` of them, part w the splits w, w + WPH, ..., then the warps in order. The
// maxima and sums are read a lane each, so that the partial outputs' loads depend on
// nothing and overlap.
template <int WPH>
__device__ __forceinline__ void join_splits(const float* base, int n, int dh, int part, int warp, int lane, float (&so)[8][256],
                                            float (&sm)[8][2], float* out) {
    const int stride = dh + 4;
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
    if (!out) return;
    const float inv = L == 0.0f ? 0.0f : fdiv(1.0f, L);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = 4 * lane + 128 * i;
        if (d < dh)
            *reinterpret_cast<float4*>(out + d) =
                make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
    }
}

}  // namespace b2
