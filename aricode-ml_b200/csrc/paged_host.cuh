// paged_host.cuh — host-side checks shared by the entry points over the paged 8-bit KV
// cache (paged.cu, tree.cu): head sizes, the cache and the rows of a call as the kernels
// take them.
#pragma once
#include "host_checks.cuh"
#include "paged_rows.cuh"

namespace b2 {

inline const char* head_dim_bad(int dh) {
    return dh < 16 || dh > 256 || dh % 16 ? "d_head must be a multiple of 16 from 16 to 256" : nullptr;
}

constexpr int kMaxPagedHeads = 1024;
// Every CTA goes through the sequences to find its own, so that a call's time grows with
// their square: single tokens, 32 / 8 heads of 128, append and attention 0.04 and 0.07 ms for
// 512 sequences, 0.25 and 0.5 for 2048, 3.4 and 5.7 for 8192, 239 and 416 for 65536. A million
// would hold the GPU for minutes.
constexpr int kMaxSeqs = 65536;

// the cache and the rows of a call, checked; false: refused with a message
inline bool view(const char* fn, const b2_kv_pages* kv, const b2_kv_rows* rows, PagedKv& c, PagedRows& r) {
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

}  // namespace b2
