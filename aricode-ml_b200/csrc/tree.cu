// tree.cu — entry points of the trees of drafted tokens (tree.cuh): argument checks and
// launches. Device pointers in and out, caller's stream, nothing allocated, nothing
// synchronised, and nothing read from device memory on the host.
#include <algorithm>

#include "paged_host.cuh"
#include "tree.cuh"

using namespace b2;

namespace {

bool al8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

// the rows of a call, checked but for page_table; false: refused with a message
bool tree_view(const char* fn, const b2_tree_rows* t, PagedRows& r) {
    auto bad = [&](const char* why) { refuse(fn, why); return false; };
    if (!t) return bad("NULL tree");
    if (t->n_rows < 0 || t->n_seq < 0 || t->max_pages < 0 || t->max_keys < 0 || t->max_rows < 0) return bad("negative count");
    if (t->n_seq > kMaxSeqs) return bad("n_seq above 65536");
    if (t->n_rows > 0 && t->n_seq > 0 &&
        (!t->row_start || !t->kv_len || !t->seen || !al4(t->row_start) || !al4(t->kv_len) || !al8(t->seen)))
        return bad("row_start, kv_len and seen must be set, seen 8-byte aligned");
    r.row_start = t->row_start; r.kv_len = t->kv_len; r.table = t->page_table;
    r.n_seq = t->n_seq; r.max_pages = t->max_pages; r.n_rows = t->n_rows;
    return true;
}

// the same with the cache
bool tree_view(const char* fn, const b2_kv_pages* kv, const b2_tree_rows* t, PagedKv& c, PagedRows& r) {
    if (!t) return refuse(fn, "NULL tree") == B2_OK;
    const b2_kv_rows rows{t->row_start, t->kv_len, t->page_table, t->n_seq, t->max_pages, t->n_rows, t->max_keys, t->max_rows};
    return view(fn, kv, &rows, c, r) && tree_view(fn, t, r);
}

// Columns of an item: 16 where no sequence has more (one token, short chains without shared heads), else as many
// as the tensor memory and shared memory hold: 64, or 32 for d_head above 128. Items of 16 and of 64 (32), us in a captured
// graph, by the columns (row, head) that a KV head has:
//                                              16         32          48           64
//   8 sequences, 4000 keys, 32 / 8 heads of 128   51  82   72  86    86   90    111   94
//   32, 1152 keys, 32 / 8 heads of 128            53  88   76  94   107  100    125  107
//   8, 4000 keys, 32 / 8 heads of 64              47  64   66  68    82   78    107   84
//   8, 2000 keys, 16 / 4 heads of 256             39  49   57  51    66   76     84   78
// (up to 32 columns several items of 16 would be as fast or faster below d_head 256). Longer: 16 sequences of up to 60 rows
// over 4000 keys 261 and 208, 2 of 64 rows over 40 K keys, 32 / 4 heads of 64 755 and 343.
int tree_columns(const TreeAttnParams& p, int max_rows) {
    const int rows = std::min(max_rows > 0 ? std::min(max_rows, kTreeRows) : kTreeRows, p.r.n_rows);
    return rows * p.G <= 16 ? 16 : p.c.dh > 128 ? 32 : 64;
}

// Keys of a split: so many items that the last round of the GPU is nearly full, in four to eight rounds (lengths
// differ, and the host does not know them), of 256 keys at least; an item beside its keys costs about two tiles of them.
// (Powers of two, eight rounds: 40 K keys, two sequences of 64 rows of 32 / 4 heads of 64 in 640 items 429 us. Eight to
// sixteen rounds: the same 356 us instead of 320 in a captured graph; 4 of 8 rows over 20 K keys, 32 / 8 heads of 128, 143 instead of 133.
// Two to four: 320 and 127; 16 of 40 rows over 3000 keys, all of one length, 236 instead of 272; sequences of different lengths
// up to 4000 keys 208 either way. 148 SMs whatever the device has, so that the workspace is the same everywhere.)
void tree_plan(TreeAttnParams& p, int nc) {
    const long long tiles = std::max((long long)p.r.n_rows * p.G / nc, (long long)std::min(p.r.n_seq, p.r.n_rows)) * p.c.KVH;
    const long long most = std::max(1ll, std::min((p.r.cap + 255ll) / 256, 1024ll)), keys = (p.r.cap + kTreeKeys - 1ll) / kTreeKeys;
    long long best = 0;
    p.kc = kTreeKeys;
    for (int rounds = 4; rounds <= 8; ++rounds) {
        const long long n = std::max(1ll, std::min(148ll * rounds / std::max(tiles, 1ll), most));
        const long long len = std::max(1ll, (keys + n - 1) / n), splits = (keys + len - 1) / len;
        const long long cost = (tiles * splits + 147) / 148 * (len + 2);
        if (best == 0 || cost < best) {
            best = cost;
            p.kc = (int)std::min(len * kTreeKeys, 1ll << 30);
        }
    }
    p.nsplit = std::max(1, (p.r.cap - 1) / p.kc + 1);
}

// items that the call can have at most
long long tree_items(const TreeAttnParams& p, int nc) {
    return ((long long)p.r.n_rows * p.G / nc + std::min(p.r.n_seq, p.r.n_rows)) * p.c.KVH * p.nsplit;
}

size_t tree_bytes(const TreeAttnParams& p) {
    return p.nsplit > 1 ? (size_t)p.r.n_rows * p.H * p.nsplit * (p.c.dh + 4) * sizeof(float) : 0;
}

template <int DP, int NC>
cudaError_t launch_tree(const TreeAttnParams& p, cudaStream_t s) {
    auto k = tree_attn_kernel<DP, NC>;
    cudaError_t e = allow_smem<tree_attn_kernel<DP, NC>>(TreeShape<DP, NC>::Alloc);
    if (e != cudaSuccess) return e;
    e = launch_ex(k, dim3((unsigned)std::min<long long>(tree_items(p, NC), sm_count())), dim3(TreeShape<DP, NC>::Threads), TreeShape<DP, NC>::Alloc, s, true, p);
    if (e != cudaSuccess || p.nsplit == 1) return e;
    if (p.nsplit <= 8) return launch_ex(tree_join_kernel<1>, dim3((unsigned)p.r.n_rows, (unsigned)((p.H + 7) / 8)), dim3(256), 0, s, true, p);
    return launch_ex(tree_join_kernel<8>, dim3((unsigned)p.r.n_rows, (unsigned)p.H), dim3(256), 0, s, true, p);
}

// Splits of a row's logits: enough CTAs for the GPU, at least 2048 logits each.
int accept_splits(const b2_tree_rows* t, int vocab) {
    const int want = std::max(1, 4 * 148 / std::max(t->n_rows, 1));
    return std::max(1, std::min(want, (vocab + 2047) / 2048));
}

size_t accept_bytes(const b2_tree_rows* t, int splits) {
    return ((size_t)t->n_rows * splits + t->n_seq) * 8 + (size_t)t->n_rows * 4;
}

}  // namespace

extern "C" {

size_t b2_attn_tree_i8_workspace(const b2_kv_pages* kv, const b2_tree_rows* tree, int n_heads) {
    TreeAttnParams p{};
    if (!tree_view("b2_attn_tree_i8_workspace", kv, tree, p.c, p.r) || n_heads <= 0 || n_heads % kv->n_kv_heads) return 0;
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return 0;
    p.H = n_heads; p.G = n_heads / kv->n_kv_heads;
    tree_plan(p, tree_columns(p, tree->max_rows));
    return tree_bytes(p);
}

int b2_attn_tree_i8(const b2_kv_pages* kv, const b2_tree_rows* tree, const float* q, int64_t ldq, const float* k,
                    int64_t ldk, const float* v, int64_t ldv, float* out, int64_t ldo, int n_heads, void* workspace,
                    size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "b2_attn_tree_i8";
    TreeAttnParams p{};
    if (!tree_view(fn, kv, tree, p.c, p.r)) return B2_E_INVALID;
    if (n_heads <= 0 || n_heads > kMaxPagedHeads || n_heads % kv->n_kv_heads)
        return refuse(fn, "n_heads must be a multiple of n_kv_heads up to 1024");
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return B2_OK;
    const int64_t width = (int64_t)n_heads * kv->d_head, kvw = (int64_t)kv->n_kv_heads * kv->d_head;
    if (!rows_ok(q, ldq, width) || !rows_ok(k, ldk, kvw) || !rows_ok(v, ldv, kvw) || !rows_ok(out, ldo, width))
        return refuse(fn, "q, k, v and out: 16-byte aligned, row strides a multiple of 4 that hold a row");
    if (!al4(err)) return refuse(fn, "err must be 4-byte aligned");
    const Span o{out, ldo, width};
    if (overlap({q, ldq, width}, o, p.r.n_rows) || overlap({k, ldk, kvw}, o, p.r.n_rows) || overlap({v, ldv, kvw}, o, p.r.n_rows))
        return refuse(fn, "out must not overlap q, k or v");
    if ((int64_t)p.r.n_rows * n_heads > (1ll << 26)) return refuse(fn, "more than 2^26 (row, head) pairs");
    p.seen = reinterpret_cast<const long long*>(tree->seen);
    p.q = q; p.k = k; p.v = v; p.out = out;
    p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
    p.H = n_heads; p.G = n_heads / kv->n_kv_heads; p.err = err;
    const int nc = tree_columns(p, tree->max_rows);
    tree_plan(p, nc);
    if (tree_items(p, nc) >= (1ll << 31)) return refuse(fn, "too many (row, head, split) pieces for one call: use fewer rows or a smaller max_keys");
    const size_t need = tree_bytes(p);
    if (need && (!workspace || !al16(workspace) || workspace_bytes < need))
        return refuse(fn, "needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    const int64_t n = p.r.n_rows, codes = (int64_t)kv->n_pages * kv->n_kv_heads * kv->page_size * kv->d_head, scales = codes / kv->d_head / kKvBlock * 4;
    const Bytes read[] = {{kv->k, codes}, {kv->v, codes}, {kv->k_scale, scales}, {kv->v_scale, scales},
                          {tree->row_start, 4 * (p.r.n_seq + 1ll)}, {tree->kv_len, 4ll * p.r.n_seq},
                          {tree->page_table, 4ll * p.r.n_seq * p.r.max_pages}, {tree->seen, 8 * n}};
    const Bytes rows[] = {rows_bytes(q, ldq, width, n, 4), rows_bytes(k, ldk, kvw, n, 4), rows_bytes(v, ldv, kvw, n, 4),
                          rows_bytes(out, ldo, width, n, 4)};
    const Bytes ws = {workspace, (int64_t)need};
    if (touch(rows[3], read)) return refuse(fn, "out overlaps the cache or the tree");
    if (touch(ws, read) || touch(ws, rows)) return refuse(fn, "the workspace overlaps an input or out");
    p.part = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p.c.dh <= 64) return status(fn, nc == 16 ? launch_tree<64, 16>(p, s) : launch_tree<64, 64>(p, s));
    if (p.c.dh <= 128) return status(fn, nc == 16 ? launch_tree<128, 16>(p, s) : launch_tree<128, 64>(p, s));
    return status(fn, nc == 16 ? launch_tree<256, 16>(p, s) : launch_tree<256, 32>(p, s));
}

size_t b2_tree_accept_workspace(const b2_tree_rows* tree, int vocab) {
    PagedRows r{};
    if (!tree_view("b2_tree_accept_workspace", tree, r) || vocab <= 0 || r.n_rows == 0 || r.n_seq == 0) return 0;
    return accept_bytes(tree, accept_splits(tree, vocab));
}

int b2_tree_accept(const b2_tree_rows* tree, const float* logits, int64_t ld, int vocab, const int32_t* tokens,
                   int32_t* kept_start, int32_t* kept_len, int32_t* kept_rows, int32_t* kept_ids, void* workspace,
                   size_t workspace_bytes, int32_t* err, void* stream) {
    const char* fn = "b2_tree_accept";
    TreeAcceptParams p{};
    if (!tree_view(fn, tree, p.r)) return B2_E_INVALID;
    if (vocab <= 0 || vocab > (1 << 30) || ld < vocab) return refuse(fn, "vocab must be 1 to 2^30, ld hold a row");
    const int64_t n = p.r.n_rows, ns = p.r.n_seq;
    const bool none = n == 0 || ns == 0;                           // no paths: sums and lengths alone
    if (none && (!tree->row_start || (ns && !tree->kv_len))) return B2_OK;
    if (!kept_start || (ns && !kept_len) || !al4(kept_start) || !al4(kept_len) || !al4(err) ||
        (none ? !al4(tree->row_start) || !al4(tree->kv_len)
              : !logits || !tokens || !kept_rows || !kept_ids || !al4(logits) || !al4(tokens) || !al4(kept_rows) || !al4(kept_ids)))
        return refuse(fn, "logits, tokens and the kept arrays must be set, 4-byte aligned");
    auto words = [](const void* x, int64_t n) { return Span{static_cast<const float*>(x), n, n}; };
    const Span outs[4] = {words(kept_start, ns + 1), words(kept_len, ns), words(kept_rows, n), words(kept_ids, n)};
    const Span ins[4] = {words(tree->row_start, ns + 1), words(tree->kv_len, ns), words(tree->seen, 2 * n), words(tokens, n)};
    for (int i = 0; i < (none ? 2 : 4); ++i) {
        bool bad = !none && overlap({logits, ld, vocab}, {outs[i].p, 0, outs[i].width}, n);
        for (int j = 0; j < (none ? 2 : 4); ++j)
            bad = bad || (j > i && overlap(outs[i], outs[j], 1)) || (overlap(outs[i], ins[j], 1) && !(i == 1 && j == 1 && same(outs[i], ins[j])));
        if (bad) return refuse(fn, "a kept array overlaps an input (other than kept_len being kv_len) or another one");
    }
    p.kept_start = kept_start; p.kept_len = kept_len; p.err = err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (none) return status(fn, launch_ex(tree_none_kernel, dim3((unsigned)(ns / 256 + 1)), dim3(256), 0, s, true, p));
    p.splits = accept_splits(tree, vocab);
    const size_t need = accept_bytes(tree, p.splits);
    if (!workspace || !al16(workspace) || workspace_bytes < need)
        return refuse(fn, "needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    const Bytes ws = {workspace, (int64_t)need}, rows = rows_bytes(logits, ld, vocab, n, 4);
    bool bad = touch(ws, rows);
    for (int i = 0; i < 4; ++i) bad = bad || touch(ws, {outs[i].p, 4 * outs[i].width}) || touch(ws, {ins[i].p, 4 * ins[i].width});
    if (bad) return refuse(fn, "the workspace overlaps an input or a kept array");
    p.seen = reinterpret_cast<const long long*>(tree->seen);
    p.logits = logits; p.ld = ld; p.vocab = vocab;
    p.chunk = ((vocab + p.splits - 1) / p.splits + 3) / 4 * 4;
    p.tokens = tokens; p.kept_rows = kept_rows; p.kept_ids = kept_ids;
    p.best = static_cast<unsigned long long*>(workspace);
    p.paths = p.best + (size_t)p.r.n_rows * p.splits;
    p.ids = reinterpret_cast<int*>(p.paths + p.r.n_seq);
    cudaError_t e = launch_ex(tree_argmax_kernel, dim3((unsigned)p.r.n_rows * p.splits), dim3(256), 0, s, true, p);
    if (e == cudaSuccess) e = launch_ex(tree_path_kernel, dim3(1), dim3(1024), 0, s, true, p);
    return status(fn, e);
}

}  // extern "C"
