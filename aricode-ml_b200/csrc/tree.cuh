// tree.cuh — trees of drafted tokens: acceptance of the path that the logits confirm
// (sm_100a). A call's rows are ragged as in paged_rows.cuh, except that kv_len counts the
// cached keys alone. Up to 64 rows a sequence, so that what a row sees of them is one 64-bit
// word. (The attention is in tree_attn.cuh.)
#pragma once
#include "tree_attn.cuh"

namespace b2 {

// A logit and its index as one word, so that the largest word is the largest logit's first
// index: the value as an unsigned number in its order (a NaN below all, -0 as +0), above the
// complement of the index.
__device__ __forceinline__ unsigned long long logit_word(float x, unsigned i) {
    const unsigned b = __float_as_uint(fadd(x, 0.0f)), o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)(x == x ? o : 0u) << 32 | (0xffffffffu - i);
}

struct TreeAcceptParams {
    PagedRows r;
    const long long* seen;
    const float* logits;     // [n_rows][ld]
    long long ld;
    int vocab, splits, chunk;   // a split: chunk logits (a multiple of 4)
    const int* tokens;
    int* kept_start;
    int* kept_len;
    int* kept_rows;
    int* kept_ids;
    unsigned long long* best;   // [n_rows][splits]
    unsigned long long* paths;  // [n_seq]
    int* ids;                   // [n_rows]
    int* err;
};

// The largest word of a row's split: CTA row * splits + split. Bound by memory (730 rows of 50257 logits: 28 us,
// 22 at 6.56 TB/s).
static __global__ void __launch_bounds__(256) tree_argmax_kernel(const __grid_constant__ TreeAcceptParams p) {
    __shared__ unsigned long long sb[8];
    after_previous();
    const int row = blockIdx.x / p.splits, split = blockIdx.x % p.splits, tid = threadIdx.x;
    if (row >= min(p.r.row_start[p.r.n_seq], p.r.n_rows)) return;      // rows of no sequence
    const float* x = p.logits + (size_t)row * p.ld;
    const int i0 = split * p.chunk, i1 = min(i0 + p.chunk, p.vocab);
    unsigned long long b = 0ull;
    // from the first 16-byte boundary on four at a time
    const int head = min(i0 + (int)((16 - (reinterpret_cast<uintptr_t>(x + i0) & 15)) / 4 & 3), i1), body = head + (i1 - head) / 4 * 4;
    if (i0 + tid < head) b = logit_word(x[i0 + tid], i0 + tid);
    if (body + tid < i1) b = max(b, logit_word(x[body + tid], body + tid));
#pragma unroll 4
    for (int i = head + 4 * tid; i < body; i += 1024) {
        const float4 v = *reinterpret_cast<const float4*>(x + i);
        b = max(max(b, max(logit_word(v.x, i), logit_word(v.y, i + 1))), max(logit_word(v.z, i + 2), logit_word(v.w, i + 3)));
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    if ((tid & 31) == 0) sb[tid >> 5] = b;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) b = max(b, sb[w]);
        // logits[0] NaN: the comparisons of the greedy choice leave 0
        if (split == 0 && x[0] != x[0]) b = 0xffffffffffffffffull;
        p.best[(size_t)row * p.splits + split] = b;
    }
}

// A call without rows: paths of nothing.
static __global__ void __launch_bounds__(256) tree_none_kernel(const __grid_constant__ TreeAcceptParams p) {
    after_previous();
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s > p.r.n_seq) return;
    p.kept_start[s] = 0;
    if (s == p.r.n_seq) return;
    p.kept_len[s] = p.r.kv_len[s];
    if (p.r.row_start[s + 1] < p.r.row_start[s]) set_err(p.err, B2_DEV_ERR_BAD_ROWS);
}

// The paths: one CTA, a warp a sequence at a time, two rows a lane; then the sums of their
// lengths, and the kept rows in order. A path's rows ascend, so a path is a 64-bit word. Bound by latency
// (48 sequences: 8.5 us).
static __global__ void __launch_bounds__(1024) tree_path_kernel(const __grid_constant__ TreeAcceptParams p) {
    __shared__ int sums[32];
    after_previous();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int live = min(p.r.row_start[p.r.n_seq], p.r.n_rows);    // rows that have a largest word
    for (int s = warp; s < p.r.n_seq; s += 32) {
        SeqRows q = seq_rows(p.r, s);
        if (p.r.row_start[s + 1] < p.r.row_start[s] && lane == 0) set_err(p.err, B2_DEV_ERR_BAD_ROWS);
        if (q.len > kTreeRows && lane == 0) set_err(p.err, B2_DEV_ERR_TOO_MANY);
        unsigned long long path = 0ull;
        const bool tree = q.len <= kTreeRows;
        q.len = min(q.len, live - q.a);                        // (less only where a start falls, which is flagged)
        if (q.len > 0 && tree) {
            int id[2], parent[2], token[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = lane + 32 * u, row = q.a + j;
                id[u] = parent[u] = token[u] = -1;
                if (j >= q.len) continue;
                const unsigned long long* best = p.best + (size_t)row * p.splits;
                unsigned long long b = best[0];
                for (int i = 1; i < p.splits; ++i) b = max(b, best[i]);
                id[u] = (int)(0xffffffffu - (unsigned)b);
                p.ids[row] = id[u];
                const unsigned long long before = (unsigned long long)p.seen[row] & ((1ull << j) - 1);
                parent[u] = 63 - __clzll((long long)before);
                token[u] = p.tokens[row];
            }
            for (int at = 0; at >= 0;) {
                path |= 1ull << at;
                const int want = __shfl_sync(0xffffffffu, at < 32 ? id[0] : id[1], at & 31);
                const unsigned lo = __ballot_sync(0xffffffffu, parent[0] == at && token[0] == want);
                const unsigned hi = __ballot_sync(0xffffffffu, parent[1] == at && token[1] == want);
                at = lo ? __ffs(lo) - 1 : hi ? __ffs(hi) + 31 : -1;
            }
        }
        if (lane == 0) p.paths[s] = path;
    }
    __syncthreads();
    // sums of the lengths, 1024 sequences at a time
    int base = 0;
    for (int s0 = 0; s0 < p.r.n_seq; s0 += 1024) {
        const int s = s0 + tid;
        const unsigned long long path = s < p.r.n_seq ? p.paths[s] : 0ull;
        const int n = __popcll(path);
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int before = base, total = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        __syncthreads();
        if (s < p.r.n_seq) {
            // (row ranges that overlap could keep more rows than there are)
            const int end = min(before + incl, p.r.n_rows), a = seq_rows(p.r, s).a;
            int at = min(end, before + incl - n);
            if (s == 0) p.kept_start[0] = 0;
            p.kept_start[s + 1] = end;
            p.kept_len[s] = p.r.kv_len[s] + end - at;
            for (unsigned long long rest = path; rest && at < end; rest &= rest - 1, ++at) {
                const int row = a + __ffsll((long long)rest) - 1;
                p.kept_rows[at] = row;
                p.kept_ids[at] = p.ids[row];
            }
        }
        base += total;
    }
}

}  // namespace b2
