"""The trees of drafted tokens and the group-scaled 4-bit products without a GPU: refusals come before a launch, struct
layouts are those of include/b2dec.h, and the host-side helpers."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
A = 1 << 20                      # stands for an aligned device address: a refused call touches none


def pages(rt, **kw):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, page_size=16, n_kv_heads=2, d_head=64)
    f.update(kw)
    return rt._KvPages(*(f[n] for n, _ in rt._KvPages._fields_))


def tree(rt, **kw):
    f = dict(row_start=A, kv_len=A, page_table=A, seen=A, n_seq=2, max_pages=3, n_rows=5, max_keys=0, max_rows=0)
    f.update(kw)
    return rt._TreeRows(*(f[n] for n, _ in rt._TreeRows._fields_))


def rows(rt, **kw):
    f = dict(row_start=A, kv_len=A, page_table=A, n_seq=2, max_pages=3, n_rows=5, max_keys=0, max_rows=0)
    f.update(kw)
    return rt._KvRows(*(f[n] for n, _ in rt._KvRows._fields_))


def attend(rt, kv, t, **kw):
    a = dict(q=A, ldq=256, k=2 * A, ldk=128, v=3 * A, ldv=128, out=4 * A, ldo=256, n_heads=4, ws=5 * A, ws_bytes=1 << 40, err=None)
    a.update(kw)
    return rt.lib().b2_attn_tree_i8(C.addressof(kv) if kv else None, C.addressof(t) if t else None, *a.values(), None)


def accept(rt, t, **kw):
    a = dict(logits=2 * A, ld=100, vocab=100, tokens=3 * A, start=4 * A, kv_len=5 * A, rows=6 * A, ids=7 * A, ws=8 * A, ws_bytes=1 << 40,
             err=None)
    a.update(kw)
    return rt.lib().b2_tree_accept(C.addressof(t) if t else None, *a.values(), None)


def append(rt, kv, r, **kw):
    a = dict(index=A, n_src=9, k=A, ldk=128, v=A, ldv=128, k_gain=None, eps=1e-5, table=None, table_rows=0, err=None)
    a.update(kw)
    return rt.lib().b2_kv_append_kept_i8(C.addressof(kv) if kv else None, C.addressof(r) if r else None, *a.values(), None)


def gemv(rt, **kw):
    a = dict(W=A, ld=64, scale=A, lds=1, bf16=0, group=128, X=2 * A, ldx=128, bias=None, Y=3 * A, ldy=7, m=7, n=128, T=3, ws=4 * A,
             ws_bytes=1 << 40)
    a.update(kw)
    return rt.lib().b2_gemv_i4_groups(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 8), dict(k_scale=None), dict(n_pages=0), dict(page_size=48),
                                 dict(n_kv_heads=0), dict(d_head=72), dict(d_head=272)])
def test_bad_caches_are_refused(pkg, bad):
    rt = pkg.runtime
    assert attend(rt, pages(rt, **bad), tree(rt)) == -1 and rt.last_error().startswith("b2_attn_tree_i8")
    assert append(rt, pages(rt, **bad), rows(rt)) == -1 and rt.last_error().startswith("b2_kv_append_kept_i8")


@pytest.mark.parametrize("bad", [dict(row_start=None), dict(kv_len=None), dict(seen=None), dict(seen=A + 4), dict(kv_len=A + 1),
                                 dict(n_seq=-1), dict(n_rows=-1), dict(max_pages=-1), dict(max_keys=-1), dict(max_rows=-1),
                                 dict(n_seq=65537)])
def test_bad_trees_are_refused(pkg, bad):
    rt = pkg.runtime
    assert attend(rt, pages(rt), tree(rt, **bad)) == -1
    assert accept(rt, tree(rt, **bad)) == -1 and rt.last_error().startswith("b2_tree_accept")


@pytest.mark.parametrize("bad", [dict(page_table=None), dict(max_pages=1 << 27)])
def test_bad_page_tables_are_refused(pkg, bad):
    """By the attention alone: acceptance reads no pages."""
    assert attend(pkg.runtime, pages(pkg.runtime), tree(pkg.runtime, **bad)) == -1


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=A + 4), dict(k=A + 8), dict(ldq=252),
                                 dict(ldk=126), dict(ldv=124), dict(ldo=250), dict(n_heads=3), dict(n_heads=0), dict(n_heads=2048),
                                 dict(err=A + 1), dict(out=A), dict(out=2 * A + 16), dict(out=3 * A - 4 * 1024)])
def test_bad_attention_is_refused(pkg, bad):
    assert attend(pkg.runtime, pages(pkg.runtime), tree(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(logits=None), dict(logits=A + 2), dict(ld=99), dict(vocab=0), dict(vocab=-5), dict(tokens=None),
                                 dict(start=None), dict(kv_len=A + 1), dict(rows=None), dict(ids=None), dict(ws=None), dict(ws=A + 8),
                                 dict(ws_bytes=3), dict(err=A + 2)])
def test_bad_acceptance_is_refused(pkg, bad):
    assert accept(pkg.runtime, tree(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(start=A), dict(kv_len=A + 4), dict(rows=3 * A), dict(ids=3 * A + 16), dict(rows=7 * A - 4),
                                 dict(ids=6 * A + 4), dict(start=5 * A - 8), dict(rows=A), dict(ids=2 * A + 1600), dict(kv_len=4 * A + 8)])
def test_kept_arrays_that_overlap_are_refused(pkg, bad):
    """row_start, kv_len and seen at A; logits, tokens and the kept arrays from 2 A on: 5 rows, 2 sequences."""
    assert accept(pkg.runtime, tree(pkg.runtime), **bad) == -1
    assert "overlaps" in pkg.runtime.last_error()


@pytest.mark.parametrize("bad", [dict(index=None), dict(index=A + 2), dict(n_src=-1), dict(k=None), dict(v=A + 4), dict(ldk=124),
                                 dict(ldv=130), dict(k_gain=A + 4), dict(table=A), dict(table=A + 8, table_rows=4),
                                 dict(k_gain=A, eps=-1.0), dict(k_gain=A, eps=float("nan")), dict(err=A + 1)])
def test_bad_kept_appends_are_refused(pkg, bad):
    assert append(pkg.runtime, pages(pkg.runtime), rows(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(W=None), dict(W=A + 8), dict(ld=48), dict(ld=72), dict(n=129), dict(scale=None), dict(scale=A + 2),
                                 dict(scale=A + 1, bf16=1), dict(lds=0), dict(group=16), dict(group=256), dict(group=0), dict(X=None),
                                 dict(X=A + 2), dict(Y=None), dict(ldx=127), dict(ldy=6), dict(bias=A + 1), dict(m=-1), dict(n=0),
                                 dict(T=-1), dict(Y=2 * A), dict(Y=2 * A + 128 * 4)])
def test_bad_products_are_refused(pkg, bad):
    rt = pkg.runtime
    assert gemv(rt, **bad) == -1 and rt.last_error().startswith("b2_gemv_i4_groups")


@pytest.mark.parametrize("big", [(1 << 31) - 1, (1 << 31) - 65535])
def test_products_beyond_32_bits_are_refused(pkg, big):
    """Sizes whose last tile or part would be counted past 2^31."""
    rt = pkg.runtime
    for kw in (dict(n=big, ld=1 << 30, lds=1 << 26, ldx=1 << 31), dict(m=big, ldy=1 << 31), dict(T=big), dict(T=1, n=big, ld=1 << 30, lds=1 << 26, ldx=1 << 31)):
        assert gemv(rt, **kw) == -1 and "at most" in rt.last_error()
    assert rt.lib().b2_gemv_i4_groups_workspace(big, 128) == 0 and rt.lib().b2_gemv_i4_groups_workspace(3, big) == 0


@pytest.mark.parametrize("bad", [dict(Y=A), dict(Y=A + 7 * 64 - 4, scale=5 * A), dict(W=5 * A, Y=A + 6 * 4), dict(W=5 * A, scale=6 * A, bias=3 * A + 4),
                                 dict(Y=4 * A), dict(Y=4 * A - 4), dict(ws=A), dict(ws=2 * A + 2 * 128 * 4), dict(ws=3 * A + 80),
                                 dict(ws=5 * A, bias=5 * A + 16)])
def test_products_whose_memory_overlaps_are_refused(pkg, bad):
    """W, scale at A, X at 2 A, Y at 3 A, the workspace at 4 A: 7 rows, 128 columns, 3 vectors."""
    assert gemv(pkg.runtime, **bad) == -1 and "overlaps" in pkg.runtime.last_error()


@pytest.mark.parametrize("cache", [dict(k=4 * A), dict(v=4 * A + 4096), dict(k=4 * A - 8192 + 16), dict(k_scale=4 * A + 64), dict(v_scale=4 * A - 28)])
def test_attention_into_the_cache_is_refused(pkg, cache):
    """out at 4 A: 5 rows of 256; 4 pages of 16 x 2 x 64 codes, 8 scales each."""
    rt = pkg.runtime
    assert attend(rt, pages(rt, **cache), tree(rt)) == -1 and "out overlaps" in rt.last_error()


@pytest.mark.parametrize("t", [dict(row_start=4 * A + 8), dict(kv_len=4 * A - 4), dict(page_table=4 * A + 16), dict(seen=4 * A - 32)])
def test_attention_into_the_tree_is_refused(pkg, t):
    rt = pkg.runtime
    assert attend(rt, pages(rt), tree(rt, **t)) == -1 and "out overlaps" in rt.last_error()


@pytest.mark.parametrize("at", [A, 2 * A + 16, 3 * A, 4 * A + 32, A + 8000])
def test_a_workspace_over_what_a_call_uses_is_refused(pkg, at):
    """Calls that need one: attention of many pages, acceptance."""
    rt = pkg.runtime
    t = tree(rt, max_pages=64)
    assert rt.lib().b2_attn_tree_i8_workspace(C.addressof(pages(rt)), C.addressof(t), 4) > 0
    assert attend(rt, pages(rt), t, ws=at) == -1 and "workspace overlaps" in rt.last_error()
    kept = dict(start=4 * A, kv_len=5 * A, rows=6 * A, ids=7 * A)
    for ws in (2 * A + 48, 3 * A, 4 * A, 5 * A, 6 * A - 16, 7 * A + 16, A):
        assert accept(rt, tree(rt), ws=ws, **kept) == -1 and "workspace overlaps" in rt.last_error()


def test_nothing_to_do_is_no_error(pkg):
    rt = pkg.runtime
    none = dict(row_start=None, kv_len=None, page_table=None, seen=None, max_pages=0)
    for t in (tree(rt, n_rows=0, **none), tree(rt, n_seq=0, **none)):
        assert attend(rt, pages(rt), t, q=None, k=None, v=None, out=None, ws=None) == 0
        assert accept(rt, t, logits=None, ws=None) == 0
        assert rt.lib().b2_attn_tree_i8_workspace(C.addressof(pages(rt)), C.addressof(t), 4) == 0
        assert rt.lib().b2_tree_accept_workspace(C.addressof(t), 100) == 0
    assert append(rt, pages(rt), rows(rt, n_rows=0, row_start=None, kv_len=None), k=None) == 0
    assert gemv(rt, m=0, W=None) == 0 and gemv(rt, T=0, X=None) == 0


@pytest.mark.parametrize("bad", [dict(start=None), dict(kv_len=None), dict(start=4 * A + 2), dict(kv_len=A + 6), dict(err=A + 1),
                                 dict(start=A), dict(start=A + 8), dict(kv_len=A + 4), dict(kv_len=4 * A + 8)])
def test_bad_acceptance_of_no_rows_is_refused(pkg, bad):
    """Sums and lengths are written then too: 2 sequences, row_start and kv_len at A."""
    a = dict(logits=None, tokens=None, rows=None, ids=None, ws=None)
    assert accept(pkg.runtime, tree(pkg.runtime, n_rows=0), **{**a, **bad}) == -1
    assert accept(pkg.runtime, tree(pkg.runtime, n_rows=0, row_start=A + 2), **a) == -1


def test_null_structs_are_refused(pkg):
    rt = pkg.runtime
    assert attend(rt, None, tree(rt)) == -1 and attend(rt, pages(rt), None) == -1 and accept(rt, None) == -1
    assert append(rt, None, rows(rt)) == -1 and append(rt, pages(rt), None) == -1


def test_workspace_of_refused_shapes_is_zero(pkg):
    rt = pkg.runtime
    L = rt.lib()
    assert L.b2_attn_tree_i8_workspace(None, None, 4) == 0
    assert L.b2_attn_tree_i8_workspace(C.addressof(pages(rt, d_head=8)), C.addressof(tree(rt)), 4) == 0
    assert L.b2_attn_tree_i8_workspace(C.addressof(pages(rt)), C.addressof(tree(rt)), 3) == 0
    assert L.b2_tree_accept_workspace(None, 100) == 0 and L.b2_tree_accept_workspace(C.addressof(tree(rt)), 0) == 0
    assert L.b2_gemv_i4_groups_workspace(0, 128) == 0 and L.b2_gemv_i4_groups_workspace(4, -1) == 0


def test_struct_layout_is_the_headers(pkg, tmp_path):
    src = tmp_path / "s.cpp"
    names = [n for n, _ in pkg.runtime._TreeRows._fields_]
    src.write_text('#include <cstddef>\n#include <cstdio>\n#include "b2dec.h"\nint main() { printf("%zu %d %d %d", sizeof(b2_tree_rows), '
                   'B2_TREE_ROWS, B2_TREE_BAD_ROW, B2_TREE_TOO_MANY);\n'
                   + "".join(f'printf(" %zu", offsetof(b2_tree_rows, {n}));\n' for n in names) + "}\n")
    subprocess.run(["g++", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    rt = pkg.runtime
    assert got[:4] == [C.sizeof(rt._TreeRows), rt.TREE_ROWS, 6, 7] and {6, 7} <= set(rt.TREE_ERRORS)
    assert got[4:] == [getattr(rt._TreeRows, n).offset for n in names]


def test_what_rows_of_a_tree_see(pkg):
    seen = pkg.runtime.tree_seen
    assert seen([]) == [] and seen([-1]) == [1] and seen([-1, 0, 1]) == [1, 3, 7]
    assert seen([-1, 0, 0, 1, 2, -1]) == [1, 0b11, 0b101, 0b1011, 0b10101, 0b100000]
    assert seen([-1] + list(range(63)))[-1] == -1                   # all 64 bits
    for bad in ([0], [-1, 1], [-1, -2], [-1] * 65):
        with pytest.raises(pkg.runtime.B2Error):
            seen(bad)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 31, 128, 130, 257])
def test_group_quantiser(pkg, group, n):
    """Codes and scales of each group are those of the per-row quantiser on that group alone."""
    W = np.random.default_rng(n).standard_normal((5, n)).astype(np.float32)
    W[1] = 0
    packed, scales = pkg.pack.quantize_groups_i4(W, group)
    assert packed.shape == (5, (n + 31) // 32 * 16) and scales.shape == (5, -(-n // group)) and scales.dtype == np.float32
    codes = np.stack((packed & 15, packed >> 4), -1).reshape(5, -1).astype(np.int8)
    codes = (codes ^ 8) - 8
    assert not codes[:, n:].any()
    for g in range(0, n, group):
        top = np.abs(W[:, g:g + group]).max(1)
        assert np.array_equal(scales[:, g // group], (top / 7).astype(np.float32))
        step = np.where(top > 0, scales[:, g // group], 1)[:, None]
        assert np.array_equal(codes[:, g:min(g + group, n)], np.round(W[:, g:g + group] / step).clip(-8, 7).astype(np.int8))
    with pytest.raises(pkg.pack.PackError):
        pkg.pack.quantize_groups_i4(W, 16)
