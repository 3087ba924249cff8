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
    return 0;
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
    return status(fn, launch_ex(tree_attn_kernel, dim3((unsigned)p.r.n_rows, (unsigned)((n_heads + 7) / 8)), dim3(256), 0,
                                static_cast<cudaStream_t>(stream), true, p));
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
    if (p.r.n_rows == 0 || p.r.n_seq == 0) return B2_OK;
    if (!logits || !tokens || !kept_start || !kept_len || !kept_rows || !kept_ids || !al4(logits) || !al4(tokens) ||
        !al4(kept_start) || !al4(kept_len) || !al4(kept_rows) || !al4(kept_ids) || !al4(err))
        return refuse(fn, "logits, tokens and the kept arrays must be set, 4-byte aligned");
    p.splits = accept_splits(tree, vocab);
    const size_t need = accept_bytes(tree, p.splits);
    if (!workspace || !al16(workspace) || workspace_bytes < need)
        return refuse(fn, "needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    p.seen = reinterpret_cast<const long long*>(tree->seen);
    p.logits = logits; p.ld = ld; p.vocab = vocab;
    p.chunk = ((vocab + p.splits - 1) / p.splits + 3) / 4 * 4;
    p.tokens = tokens; p.kept_start = kept_start; p.kept_len = kept_len; p.kept_rows = kept_rows; p.kept_ids = kept_ids;
    p.best = static_cast<unsigned long long*>(workspace);
    p.paths = p.best + (size_t)p.r.n_rows * p.splits;
    p.ids = reinterpret_cast<int*>(p.paths + p.r.n_seq);
    p.err = err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_ex(tree_argmax_kernel, dim3((unsigned)p.splits, (unsigned)p.r.n_rows), dim3(256), 0, s, true, p);
    if (e == cudaSuccess) e = launch_ex(tree_path_kernel, dim3(1), dim3(1024), 0, s, true, p);
    return status(fn, e);
}

}  // extern "C"
