// paged.cu — entry points of the paged 8-bit KV cache (paged.cuh): argument checks
// and launches. Device pointers in and out, caller's stream, nothing allocated,
// nothing synchronised, and nothing read from device memory on the host.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/b2dec.h"
#include "paged.cuh"

void b2_internal_set_error(const std::string& msg);   // runtime.cu

using namespace b2;

namespace {

int refuse(const char* fn, const std::string& why) {
    b2_internal_set_error(std::string(fn) + ": " + why);
    return B2_E_INVALID;
}

int status(const char* fn, cudaError_t e) {
    if (e == cudaSuccess) return B2_OK;
    b2_internal_set_error(std::string(fn) + ": " + cudaGetErrorString(e));
    return B2_E_CUDA;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool al4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// f32 rows of `width` elements, `ld` apart, read and written 16 bytes at a time
bool rows_ok(const float* p, int64_t ld, int64_t width) { return p && al16(p) && ld >= width && ld % 4 == 0; }

// f32 rows as they lie in memory
struct Span {
    const float* p;
    int64_t ld, width;
};

// whether n rows each of a and b may share an element: side by side in one buffer (the
// slices of a fused projection) they do not, and rows that interleave with other strides
// count as sharing
bool overlap(const Span& a, const Span& b, int64_t n) {
    if (!a.p || !b.p || n <= 0) return false;
    const int64_t off = ((int64_t)reinterpret_cast<intptr_t>(b.p) - (int64_t)reinterpret_cast<intptr_t>(a.p)) / 4;
    if (off >= (n - 1) * a.ld + a.width || -off >= (n - 1) * b.ld + b.width) return false;
    if (a.ld != b.ld) return true;
    const int64_t at = ((off % a.ld) + a.ld) % a.ld;               // b's column, seen from a's first one
    return at < a.width || at + b.width > a.ld;
}

bool same(const Span& a, const Span& b) { return a.p == b.p && a.ld == b.ld; }

const char* head_dim_bad(int dh) {
    return dh < 16 || dh > 256 || dh % 16 ? "d_head must be a multiple of 16 from 16 to 256" : nullptr;
}

constexpr int kMaxPagedHeads = 1024;
// Every CTA goes through the sequences to find its own, so that a call's time grows with
// their square: single tokens, 32 / 8 heads of 128, append and attention 0.04 and 0.07 ms for
// 512 sequences, 0.25 and 0.5 for 2048, 3.4 and 5.7 for 8192, 239 and 416 for 65536. A million
// would hold the GPU for minutes.
constexpr int kMaxSeqs = 65536;

// the cache and the rows of a call, checked; false: refused with a message
bool view(const char* fn, const b2_kv_pages* kv, const b2_kv_rows* rows, PagedKv& c, PagedRows& r) {
    auto bad = [&](const char* why) { refuse(fn, why); return false; };
    if (!kv || !rows) return bad("NULL cache or rows");
    if (const char* why = head_dim_bad(kv->d_head)) return bad(why);
    if (kv->n_kv_heads <= 0 || kv->n_kv_heads > kMaxPagedHeads) return bad("n_kv_heads must be 1 to 1024");
    if (kv->page_size < kKvBlock || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return bad("page_size must be a power of two from 16 to 1024");
    if (kv->n_pages <= 0) return bad("n_pages must be positive");
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !al16(kv->k) || !al16(kv->v) || !al4(kv->k_scale) ||
        !al4(kv->v_scale))
        return bad("cache pointers must be set, the codes' aligned to 16 bytes");
    if (rows->n_rows < 0 || rows->n_seq < 0 || rows->max_pages < 0) return bad("negative count");
    if (rows->n_rows > 0 && rows->n_seq > 0 &&
        (!rows->row_start || !rows->kv_len || (!rows->page_table && rows->max_pages) || !al4(rows->row_start) ||
         !al4(rows->kv_len) || !al4(rows->page_table)))
        return bad("row_start, kv_len and page_table must be set");
    if (rows->n_seq > kMaxSeqs) return bad("n_seq above 65536");
    const int64_t cap = (int64_t)rows->max_pages * kv->page_size;
    if (cap > (1 << 30)) return bad("max_pages * page_size above 2^30");
    if ((int64_t)kv->n_pages * kv->n_kv_heads * (kv->page_size / kKvBlock) >= (1ll << 31)) return bad("2^31 or more blocks in the pool");
    if (rows->max_keys < 0 || rows->max_rows < 0) return bad("negative max_keys or max_rows");
    c.k = kv->k; c.v = kv->v; c.ks = kv->k_scale; c.vs = kv->v_scale;
    c.n_pages = kv->n_pages; c.KVH = kv->n_kv_heads; c.dh = kv->d_head;
    c.page_log2 = 0;
    while ((1 << c.page_log2) < kv->page_size) ++c.page_log2;
    r.row_start = rows->row_start; r.kv_len = rows->kv_len; r.table = rows->page_table;
    r.n_seq = rows->n_seq; r.max_pages = rows->max_pages; r.n_rows = rows->n_rows;
    r.cap = rows->max_keys > 0 && rows->max_keys < cap ? rows->max_keys : (int)cap;
    return true;
}

// most (sequence, block) runs that n_rows rows in n_seq ranges can make: a range of
// L rows touches at most (L - 2) / 16 + 2 blocks, and no more than L
int run_bound(const PagedRows& r) {
    const long long by_block = (long long)r.n_rows / kKvBlock + 2ll * r.n_seq;
    return (int)(by_block < r.n_rows ? by_block : r.n_rows);
}

// lanes and float4s that hold a head vector of dh elements
#define B2_BY_HEAD_DIM(dh, CALL)                 \
    (dh) <= 16   ? CALL(4, 1)                    \
    : (dh) <= 32 ? CALL(8, 1)                    \
    : (dh) <= 64 ? CALL(16, 1)                   \
    : (dh) <= 128 ? CALL(32, 1) : CALL(32, 2)

template <int LPH, int VPL>
cudaError_t launch_norm_rope(const NormRopeParams& p, cudaStream_t s) {
    // four vectors a lane group once there is work for the whole GPU (their loads are
    // in flight together and share the table row), one before that
    const bool four = (long long)p.n_rows * (p.H + p.KVH) * LPH >= 4ll * 148 * 1024;
    const int hpu = four ? 4 : 1;
    const long long lanes = (long long)p.n_rows * ((p.H + hpu - 1) / hpu + (p.KVH + hpu - 1) / hpu) * LPH;
    const unsigned grid = (unsigned)((lanes + 255) / 256);
    return launch_ex(four ? norm_rope_kernel<LPH, VPL, 4> : norm_rope_kernel<LPH, VPL, 1>, dim3(grid), dim3(256), 0, s, true, p);
}

template <int LPH, int VPL>
cudaError_t launch_append(AppendParams p, bool queries, int max_rows, cudaStream_t s) {
    // single rows (said by the caller, or on average): one row in registers, queries along
    if (max_rows == 1 || p.r.n_rows <= p.r.n_seq) {
        p.kv_ctas = (2 * p.c.KVH + 7) / 8;
        const int y = p.kv_ctas + (queries ? (p.nr.H * LPH + 255) / 256 : 0);
        return launch_ex(kv_append_kernel<LPH, VPL, 1, 1>, dim3((unsigned)p.items, (unsigned)y), dim3(256), 0, s, true, p);
    }
    p.kv_ctas = p.c.KVH;
    cudaError_t e = launch_ex(kv_append_kernel<LPH, VPL, LPH <= 8 ? 1 : LPH / 8, 4>, dim3((unsigned)p.items, (unsigned)p.kv_ctas),
                              dim3(256), 0, s, true, p);
    if (e != cudaSuccess || !queries) return e;
    // about four units of 4 vectors a lane group
    const int y = (kKvBlock * ((p.nr.H + 3) / 4) * LPH / 4 + 255) / 256;
    return launch_ex(append_queries_kernel<LPH, VPL>, dim3((unsigned)p.items, (unsigned)y), dim3(256), 0, s, true, p);
}

// A call's sequences are of two kinds, by their columns (token, head) of a KV head, and
// each kind has a launch, left out where the caller's sizes say that none is of its kind.
// (One that finds none costs a wave of empty CTAs, 2.4 us, for every 148 that its rows might
// have needed: with max_rows = 1 a step of 64 tokens over 1152 keys takes 119 us for 32 / 32
// heads of 128, without it 125 us; 256 tokens, 32 / 4 heads of 64: 66 and 105 us.) A whole
// batch on one kernel cost more: a single token in a 128-row tile as much as 128, a prompt in
// 8-column tiles re-reads its keys 16 times as often.
//  few, up to 16 columns: 8 a CTA, or 2 where single tokens make no more (decode without
//  shared heads; beside prompts too). Small splits fill the GPU when there are few
//  rows; with long caches larger ones bound the partial results and their joining. Their
//  size is a function of the capacity alone; the columns a CTA follow the longest sequence,
//  so the last bits of a sequence's result can differ beside others.
//  many: 128 a CTA (64 for d_head above 128); keys are split only while there are too few
//  tiles for four rounds of the GPU (d_head above 128: for six tiles an SM). Against one
//  round: a sequence of 30 K keys 173 us, not 141, three of 8 K with 16 rows 72, not 52; but
//  twelve of up to 10 K 292, not 353, two of 3 K with 300 rows 177, not 206. The host does not
//  know the lengths.
constexpr int kFewCols = 16;

struct AttnPlan {
    bool few, many;
    int few_cols, many_cols;         // columns a CTA
    long long few_items, many_items; // at most
};

AttnPlan attn_plan(PagedAttnParams& p, int max_rows) {
    AttnPlan a{};
    p.G = p.H / p.c.KVH;
    const long long longest = (long long)(max_rows > 0 ? std::min(max_rows, p.r.n_rows) : p.r.n_rows) * p.G;
    a.many = longest > kFewCols;
    a.few = !a.many || (p.r.n_seq > 1 && p.G <= kFewCols);
    a.few_cols = longest <= 2 || (a.many && p.G <= 2) ? 2 : kSplitCols;
    a.many_cols = p.c.dh <= 128 ? kMmaRows : kTileRows;
    p.few = a.few ? (a.many ? kFewCols : INT32_MAX) : 0;
    p.kc_few = p.r.cap <= 1024 ? 8 : 9;
    const long long tiles = std::max(1ll, (long long)p.r.n_rows * p.H / a.many_cols), want = p.c.dh <= 128 ? 4 * 148 : 6 * 148;
    const long long splits = std::max(1ll, std::min(want / tiles, (p.r.cap + 255ll) / 256));
    p.kc_many = 8;
    while (p.kc_many < 30 && (splits << p.kc_many) < p.r.cap) ++p.kc_many;
    auto splits_at = [&](int kc_log2) { return std::max(1, (int)((p.r.cap + (1ll << kc_log2) - 1) >> kc_log2)); };
    p.nsplit_few = a.few ? splits_at(p.kc_few) : 1;
    p.nsplit_many = a.many ? splits_at(p.kc_many) : 1;
    if (a.few && a.many) {
        // a sequence of the few-row kind has at most this many rows
        const int most = kFewCols / p.G;
        if ((long long)p.r.n_seq * most < p.r.n_rows) p.few_rows = most;
        // whole prompts: only the few-row sequences beside them have splits to join
        if (p.nsplit_many == 1) p.join_rows = most;
    }
    auto items = [&](long long tiles, int kc_log2) { return tiles * p.c.KVH * splits_at(kc_log2); };
    // tiles of `cols` columns over all sequences: at most one partly filled one each
    auto tiles_of = [&](int cols) { return (long long)p.r.n_rows * p.G / cols + std::min(p.r.n_seq, p.r.n_rows); };
    long long few_tiles = tiles_of(a.few_cols), many_tiles = tiles_of(a.many_cols);
    if (a.few && a.many) {
        // sequences of the few-row kind have up to kFewCols columns each, whatever n_rows is;
        // the others have more, so a tile of theirs has at least kFewCols + 1
        few_tiles = std::min(few_tiles, (long long)p.r.n_seq * ((kFewCols + a.few_cols - 1) / a.few_cols));
        many_tiles = std::min(many_tiles, (long long)p.r.n_rows * p.G / (kFewCols + 1));
    }
    a.few_items = a.few ? items(few_tiles, p.kc_few) : 0;
    a.many_items = a.many ? items(many_tiles, p.kc_many) : 0;
    return a;
}

// bytes of the partial results of the few-row kind, then of the many-row kind. (One area
// for both, with the finer split for every row of the call, took 35 GB for 8192 rows in 9
// sequences of 32 heads of 128 at a capacity of 128 K, now 156 MB; the many-row kind's
// splits fill the GPU a few times at most, whatever the capacity is: at most 118 MB.)
struct PartBytes {
    size_t few, many;
};

PartBytes part_bytes(const PagedAttnParams& p) {
    const size_t head = (size_t)p.H * (p.c.dh + 4) * sizeof(float);
    const size_t slots = p.few_rows ? (size_t)p.r.n_seq * p.few_rows : (size_t)p.r.n_rows;
    return {p.nsplit_few > 1 ? slots * head * p.nsplit_few : 0, p.nsplit_many > 1 ? (size_t)p.r.n_rows * head * p.nsplit_many : 0};
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

cudaError_t launch_join(const PagedAttnParams& p, cudaStream_t s) {
    // up to 8 splits: a warp each (row, head), else 8
    const unsigned rows = p.join_rows ? (unsigned)(p.r.n_seq * p.join_rows) : (unsigned)p.r.n_rows;
    if (std::max(p.nsplit_few, p.nsplit_many) <= 8)
        return launch_ex(paged_attn_join_kernel<1>, dim3(rows, (unsigned)((p.H + 7) / 8)), dim3(256), 0, s, true, p);
    return launch_ex(paged_attn_join_kernel<8>, dim3(rows, (unsigned)p.H), dim3(256), 0, s, true, p);
}

template <int DP, int NC>
cudaError_t launch_few(const PagedAttnParams& p, const AttnPlan& a, cudaStream_t s) {
    using Sh = SplitShape<DP, NC>;
    auto k = paged_attn_split_kernel<DP, NC>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::Smem);
    if (e != cudaSuccess) return e;
    const long long resident = (long long)sm_count() * (DP == 256 ? 2 : DP == 128 ? 3 : 4);
    // Behind the many-row kernel not before its end: CTAs that come up while the SM is set for
    // that kernel's shared memory keep its small L1 (64 tokens, 32 / 32 heads of 128, 1152
    // keys: 152 us, now 125; 60 tokens beside a prompt of 1000: 224, now 196).
    return launch_ex(k, dim3((unsigned)std::min(a.few_items, resident)), dim3(kSplitWarps * 32), Sh::Smem, s, !a.many, p);
}

cudaError_t launch_many(const PagedAttnParams& p, const AttnPlan& a, cudaStream_t s) {
    const bool mma = p.c.dh <= 128;
    auto k = mma ? paged_attn_mma_kernel : paged_attn_tile_kernel;
    const int smem = mma ? MmaSmem::Alloc : TileShape::Smem;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return launch_ex(k, dim3((unsigned)a.many_items), dim3(mma ? kMmaThreads : 128), smem, s, true, p);
}

cudaError_t launch_attn(PagedAttnParams p, const AttnPlan& a, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    if (a.many) {
        p.lo = a.few ? kFewCols + 1 : 0; p.hi = INT32_MAX; p.kc_log2 = p.kc_many;
        e = launch_many(p, a, s);
    }
    if (e == cudaSuccess && a.few) {
        p.lo = 0; p.hi = p.few; p.kc_log2 = p.kc_few;
        const int dp = p.c.dh <= 64 ? 64 : p.c.dh <= 128 ? 128 : 256;
        e = a.few_cols == 2 ? (dp == 64 ? launch_few<64, 2>(p, a, s) : dp == 128 ? launch_few<128, 2>(p, a, s) : launch_few<256, 2>(p, a, s))
                            : (dp == 64 ? launch_few<64, 8>(p, a, s) : dp == 128 ? launch_few<128, 8>(p, a, s) : launch_few<256, 8>(p, a, s));
    }
    return e == cudaSuccess && (p.nsplit_few > 1 || p.nsplit_many > 1) ? launch_join(p, s) : e;
}

}  // namespace

extern "C" {

int b2_qk_norm_rope(const float* q, int64_t ldq, const float* k, int64_t ldk, float* q_out, int64_t ldqo, float* k_out,
                    int64_t ldko, const float* q_gain, const float* k_gain, float eps, float q_scale, const float* table,
                    int table_rows, const int32_t* pos, int n_rows, int n_heads, int n_kv_heads, int d_head,
                    int32_t* err, void* stream) {
    const char* fn = "b2_qk_norm_rope";
    if (const char* why = head_dim_bad(d_head)) return refuse(fn, why);
    if (n_rows < 0 || n_heads < 0 || n_kv_heads < 0 || n_heads > kMaxPagedHeads || n_kv_heads > kMaxPagedHeads ||
        n_heads + n_kv_heads == 0)
        return refuse(fn, "n_rows must be 0 or more, the head counts 0 to 1024 and not both 0");
    if (n_rows == 0) return B2_OK;
    if ((n_heads && (!rows_ok(q, ldq, (int64_t)n_heads * d_head) || !rows_ok(q_out, ldqo, (int64_t)n_heads * d_head))) ||
        (n_kv_heads && (!rows_ok(k, ldk, (int64_t)n_kv_heads * d_head) || !rows_ok(k_out, ldko, (int64_t)n_kv_heads * d_head))))
        return refuse(fn, "q, k and their outputs: 16-byte aligned, row strides a multiple of 4 that hold a row");
    if ((q_gain && !al16(q_gain)) || (k_gain && !al16(k_gain)) || (table && !al16(table)) || !al4(pos) || !al4(err))
        return refuse(fn, "gains and table must be 16-byte aligned, pos and err 4");
    if (table && (!pos || table_rows <= 0)) return refuse(fn, "a table needs pos and table_rows");
    if ((q_gain || k_gain) && !(eps >= 0.0f && std::isfinite(eps))) return refuse(fn, "eps must be finite and not negative");
    if ((long long)n_rows * (n_heads + n_kv_heads) >= (1ll << 26)) return refuse(fn, "2^26 or more head vectors");
    const int64_t qw = (int64_t)n_heads * d_head, kw = (int64_t)n_kv_heads * d_head;
    const Span qi{n_heads ? q : nullptr, ldq, qw}, qo{n_heads ? q_out : nullptr, ldqo, qw};
    const Span ki{n_kv_heads ? k : nullptr, ldk, kw}, ko{n_kv_heads ? k_out : nullptr, ldko, kw};
    if ((!same(qi, qo) && overlap(qi, qo, n_rows)) || (!same(ki, ko) && overlap(ki, ko, n_rows)) || overlap(qo, ki, n_rows) ||
        overlap(ko, qi, n_rows) || overlap(qo, ko, n_rows))
        return refuse(fn, "an output overlaps an input (other than being it, with its stride) or the other output");
    NormRopeParams p{};
    p.q = q; p.k = k; p.qo = q_out; p.ko = k_out;
    p.ldq = ldq; p.ldk = ldk; p.ldqo = ldqo; p.ldko = ldko;
    p.gq = q_gain; p.gk = k_gain; p.eps = eps; p.q_scale = q_scale;
    p.inv_dh = 1.0f / (float)d_head;
    p.table = table; p.table_rows = table_rows; p.pos = pos;
    p.n_rows = n_rows; p.H = n_heads; p.KVH = n_kv_heads; p.dh = d_head; p.err = err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define B2_CALL(L, V) launch_norm_rope<L, V>(p, s)
    return status(fn, B2_BY_HEAD_DIM(d_head, B2_CALL));
#undef B2_CALL
}

int b2_kv_append_i8(const b2_kv_pages* kv, const b2_kv_rows* rows, const float* k, int64_t ldk, const float* v,
                    int64_t ldv, const float* k_gain, float eps, const float* table, int table_rows, const float* q,
                    int64_t ldq, float* q_out, int64_t ldqo, const float* q_gain, float q_scale, int n_heads,
                    int32_t* err, void* stream) {
    const char* fn = "b2_kv_append_i8";
    AppendParams p{};
    if (!view(fn, kv, rows, p.c, p.r)) return B2_E_INVALID;
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return B2_OK;
    const int64_t width = (int64_t)kv->n_kv_heads * kv->d_head;
    if (!rows_ok(k, ldk, width) || !rows_ok(v, ldv, width))
        return refuse(fn, "k and v: 16-byte aligned, row strides a multiple of 4 that hold a row");
    if (q && (n_heads <= 0 || n_heads > kMaxPagedHeads)) return refuse(fn, "n_heads must be 1 to 1024");
    if (q && (!rows_ok(q, ldq, (int64_t)n_heads * kv->d_head) || !rows_ok(q_out, ldqo, (int64_t)n_heads * kv->d_head)))
        return refuse(fn, "q and q_out: 16-byte aligned, row strides a multiple of 4 that hold a row");
    if ((q_gain && !al16(q_gain)) || (k_gain && !al16(k_gain)) || (table && !al16(table)) || !al4(err))
        return refuse(fn, "gains and table must be 16-byte aligned, err 4");
    if (table && table_rows <= 0) return refuse(fn, "a table needs table_rows");
    if (q) {
        const int64_t qw = (int64_t)n_heads * kv->d_head;
        const Span qi{q, ldq, qw}, qo{q_out, ldqo, qw};
        if ((!same(qi, qo) && overlap(qi, qo, p.r.n_rows)) || overlap(qo, {k, ldk, width}, p.r.n_rows) ||
            overlap(qo, {v, ldv, width}, p.r.n_rows))
            return refuse(fn, "q_out overlaps q (other than being it, with its stride), k or v");
    }
    if ((q_gain || k_gain) && !(eps >= 0.0f && std::isfinite(eps))) return refuse(fn, "eps must be finite and not negative");
    p.k = k; p.v = v; p.ldk = ldk; p.ldv = ldv;
    p.nr.q = q; p.nr.qo = q_out; p.nr.ldq = ldq; p.nr.ldqo = ldqo;
    p.nr.gq = q_gain; p.nr.gk = k_gain; p.nr.eps = eps; p.nr.q_scale = q_scale;
    p.nr.inv_dh = 1.0f / (float)kv->d_head;
    p.nr.table = table; p.nr.table_rows = table_rows;
    p.nr.n_rows = p.r.n_rows; p.nr.H = q ? n_heads : 0; p.nr.KVH = 0; p.nr.dh = kv->d_head; p.nr.err = err;
    p.items = run_bound(p.r);
    p.err = err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define B2_CALL(L, V) launch_append<L, V>(p, q != nullptr, rows->max_rows, s)
    return status(fn, B2_BY_HEAD_DIM(kv->d_head, B2_CALL));
#undef B2_CALL
}

int b2_kv_read_i8(const b2_kv_pages* kv, const b2_kv_rows* rows, void* k_out, void* v_out, int64_t ld, int bf16,
                  int32_t* err, void* stream) {
    const char* fn = "b2_kv_read_i8";
    ReadParams p{};
    if (!view(fn, kv, rows, p.c, p.r)) return B2_E_INVALID;
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return B2_OK;
    if (!k_out || !v_out || !al16(k_out) || !al16(v_out) || ld < (int64_t)kv->n_kv_heads * kv->d_head ||
        ld % (bf16 ? 8 : 4))
        return refuse(fn, "k_out and v_out: 16-byte aligned, ld holding a row and a multiple of 16 bytes");
    if (!al4(err)) return refuse(fn, "err must be 4-byte aligned");
    const int64_t unit = bf16 ? 2 : 1, row = (int64_t)kv->n_kv_heads * kv->d_head / unit;   // in 4-byte words
    if (overlap({static_cast<const float*>(k_out), ld / unit, row}, {static_cast<const float*>(v_out), ld / unit, row}, p.r.n_rows))
        return refuse(fn, "k_out and v_out overlap");
    p.k = k_out; p.v = v_out; p.ld = ld;
    p.items = run_bound(p.r);
    p.err = err;
    const dim3 grid((unsigned)p.items, (unsigned)((2 * p.c.KVH + 7) / 8));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int dh = kv->d_head;
#define B2_CALL(L) launch_ex(bf16 ? kv_read_kernel<true, L> : kv_read_kernel<false, L>, grid, dim3(256), 0, s, true, p)
    return status(fn, dh <= 16 ? B2_CALL(2) : dh <= 32 ? B2_CALL(4) : dh <= 64 ? B2_CALL(8) : dh <= 128 ? B2_CALL(16) : B2_CALL(32));
#undef B2_CALL
}

size_t b2_attn_paged_i8_workspace(const b2_kv_pages* kv, const b2_kv_rows* rows, int n_heads) {
    PagedAttnParams p{};
    if (!view("b2_attn_paged_i8_workspace", kv, rows, p.c, p.r) || n_heads <= 0 || n_heads % kv->n_kv_heads) return 0;
    p.H = n_heads;
    attn_plan(p, rows->max_rows);
    const PartBytes part = part_bytes(p);
    return part.few + part.many;
}

int b2_attn_paged_i8(const b2_kv_pages* kv, const b2_kv_rows* rows, const float* q, int64_t ldq, float* out, int64_t ldo,
                     int n_heads, void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "b2_attn_paged_i8";
    PagedAttnParams p{};
    if (!view(fn, kv, rows, p.c, p.r)) return B2_E_INVALID;
    if (n_heads <= 0 || n_heads > kMaxPagedHeads || n_heads % kv->n_kv_heads)
        return refuse(fn, "n_heads must be a multiple of n_kv_heads up to 1024");
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return B2_OK;
    const int64_t width = (int64_t)n_heads * kv->d_head;
    if (!rows_ok(q, ldq, width) || !rows_ok(out, ldo, width))
        return refuse(fn, "q and out: 16-byte aligned, row strides a multiple of 4 that hold a row");
    if (!al4(err)) return refuse(fn, "err must be 4-byte aligned");
    if (overlap({q, ldq, width}, {out, ldo, width}, p.r.n_rows)) return refuse(fn, "out must not overlap q");
    if ((int64_t)p.r.n_rows * n_heads > (1ll << 30)) return refuse(fn, "more than 2^30 (row, head) pairs");
    p.q = q; p.ldq = ldq; p.out = out; p.ldo = ldo; p.H = n_heads; p.err = err;
    const AttnPlan plan = attn_plan(p, rows->max_rows);
    if (plan.few_items >= kMaxItems || plan.many_items >= kMaxItems)
        return refuse(fn, "too many (row, head, split) pieces for one call: use fewer rows or a smaller max_keys");
    const PartBytes part = part_bytes(p);
    const size_t need = part.few + part.many;
    if (need && (!workspace || !al16(workspace) || workspace_bytes < need))
        return refuse(fn, "needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    p.part_few = static_cast<float*>(workspace);
    p.part_many = p.part_few + part.few / sizeof(float);
    return status(fn, launch_attn(p, plan, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
