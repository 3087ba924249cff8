"""The paged 8-bit KV cache without a GPU: every refusal of its entry points comes before a launch, so it shows here,
and the struct layouts of runtime.py are those of include/b2dec.h."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
A = 1 << 20                      # stands for an aligned device address: a refused call touches none


def pages(rt, **kw):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, page_size=16, n_kv_heads=2, d_head=64)
    f.update(kw)
    return rt._KvPages(*(f[n] for n, _ in rt._KvPages._fields_))


def rows(rt, **kw):
    f = dict(row_start=A, kv_len=A, page_table=A, n_seq=2, max_pages=3, n_rows=5, max_keys=0, max_rows=0)
    f.update(kw)
    return rt._KvRows(*(f[n] for n, _ in rt._KvRows._fields_))


def append(rt, kv, r, **kw):
    a = dict(k=A, ldk=128, v=A, ldv=128, k_gain=None, eps=1e-5, table=None, table_rows=0, q=None, ldq=0, q_out=None,
             ldqo=0, q_gain=None, q_scale=1.0, n_heads=0, err=None)
    a.update(kw)
    return rt.lib().b2_kv_append_i8(C.addressof(kv) if kv else None, C.addressof(r) if r else None, *a.values(), None)


def read(rt, kv, r, **kw):
    a = dict(k=A, v=A, ld=128, bf16=0, err=None)
    a.update(kw)
    return rt.lib().b2_kv_read_i8(C.addressof(kv), C.addressof(r), *a.values(), None)


def attend(rt, kv, r, **kw):
    a = dict(q=A, ldq=256, out=2 * A, ldo=256, n_heads=4, ws=3 * A, ws_bytes=1 << 40, err=None)
    a.update(kw)
    return rt.lib().b2_attn_paged_i8(C.addressof(kv), C.addressof(r), *a.values(), None)


def norm_rope(rt, **kw):
    a = dict(q=A, ldq=256, k=A, ldk=128, qo=A, ldqo=256, ko=A, ldko=128, gq=None, gk=None, eps=1e-5, q_scale=1.0,
             table=None, table_rows=0, pos=None, n_rows=3, n_heads=4, n_kv_heads=2, d_head=64, err=None)
    a.update(kw)
    return rt.lib().b2_qk_norm_rope(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 8), dict(k_scale=None), dict(v_scale=A + 2), dict(n_pages=0),
                                 dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(n_kv_heads=0),
                                 dict(n_kv_heads=1025), dict(d_head=8), dict(d_head=72), dict(d_head=272)])
def test_bad_caches_are_refused(pkg, bad):
    rt = pkg.runtime
    kv = pages(rt, **bad)
    for call in (append, read, attend):
        assert call(rt, kv, rows(rt)) == -1
        assert rt.last_error().startswith("b2_")


@pytest.mark.parametrize("bad", [dict(row_start=None), dict(kv_len=None), dict(page_table=None), dict(kv_len=A + 1),
                                 dict(n_seq=-1), dict(n_rows=-1), dict(max_pages=-1), dict(max_pages=1 << 27),
                                 dict(max_keys=-1), dict(max_rows=-1), dict(n_seq=(1 << 20) + 1)])
def test_bad_rows_are_refused(pkg, bad):
    rt = pkg.runtime
    for call in (append, read, attend):
        assert call(rt, pages(rt), rows(rt, **bad)) == -1


def test_null_structs_are_refused(pkg):
    rt = pkg.runtime
    assert append(rt, None, rows(rt)) == -1 and append(rt, pages(rt), None) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 4), dict(ldk=124), dict(ldv=130), dict(k_gain=A + 4),
                                 dict(table=A), dict(table=A + 8, table_rows=4), dict(k_gain=A, eps=-1.0),
                                 dict(k_gain=A, eps=float("nan")), dict(q=A, n_heads=0),
                                 dict(q=A, n_heads=4, ldq=256), dict(q=A, n_heads=4, ldq=252, q_out=A, ldqo=256),
                                 dict(q=A, n_heads=4, ldq=256, q_out=A + 4, ldqo=256), dict(err=A + 1)])
def test_bad_appends_are_refused(pkg, bad):
    assert append(pkg.runtime, pages(pkg.runtime), rows(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 8), dict(ld=127), dict(ld=130), dict(ld=132, bf16=1), dict(err=A + 2)])
def test_bad_reads_are_refused(pkg, bad):
    assert read(pkg.runtime, pages(pkg.runtime), rows(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(q=A + 4), dict(ldq=255), dict(ldo=254),
                                 dict(n_heads=3), dict(n_heads=0), dict(n_heads=2048), dict(out=A), dict(err=A + 1)])
def test_bad_attention_is_refused(pkg, bad):
    assert attend(pkg.runtime, pages(pkg.runtime), rows(pkg.runtime), **bad) == -1


@pytest.mark.parametrize("bad", [dict(q=None), dict(ko=None), dict(ldq=252), dict(ldko=126), dict(q=A + 4), dict(n_rows=-1),
                                 dict(n_heads=-1), dict(n_heads=0, n_kv_heads=0), dict(n_heads=1025), dict(d_head=40),
                                 dict(d_head=0), dict(table=A, table_rows=9), dict(table=A, pos=A), dict(gq=A + 4),
                                 dict(gq=A, eps=float("inf")), dict(pos=A + 1)])
def test_bad_norm_rope_is_refused(pkg, bad):
    assert norm_rope(pkg.runtime, **bad) == -1


def test_nothing_to_do_is_no_error(pkg):
    """No rows or no sequences: no launch, whatever the row pointers are."""
    rt = pkg.runtime
    none = dict(row_start=None, kv_len=None, page_table=None, max_pages=0)
    for r in (rows(rt, n_rows=0, **none), rows(rt, n_seq=0, **none)):
        assert append(rt, pages(rt), r, k=None, v=None) == 0
        assert read(rt, pages(rt), r, k=None, v=None) == 0
        assert attend(rt, pages(rt), r, q=None, out=None) == 0
        assert rt.lib().b2_attn_paged_i8_workspace(C.addressof(pages(rt)), C.addressof(r), 4) == 0
    assert norm_rope(rt, n_rows=0, q=None, k=None, qo=None, ko=None) == 0


def test_workspace_of_refused_shapes_is_zero(pkg):
    rt = pkg.runtime
    ws = rt.lib().b2_attn_paged_i8_workspace
    assert ws(None, None, 4) == 0
    assert ws(C.addressof(pages(rt, d_head=8)), C.addressof(rows(rt)), 4) == 0
    assert ws(C.addressof(pages(rt)), C.addressof(rows(rt)), 3) == 0
    assert ws(C.addressof(pages(rt)), C.addressof(rows(rt)), -4) == 0


def test_struct_layouts_match_the_header(pkg, tmp_path):
    rt = pkg.runtime
    lines = []
    for c, py in (("b2_kv_pages", rt._KvPages), ("b2_kv_rows", rt._KvRows)):
        lines.append(f'printf("%zu ", sizeof({c}));')
        lines += [f'printf("%zu ", offsetof({c}, {n}));' for n, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "b2dec.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in (rt._KvPages, rt._KvRows):
        want += [C.sizeof(py)] + [getattr(py, n).offset for n, _ in py._fields_]
    assert got == want


def test_handles_refuse_host_tensors_and_bad_shapes(pkg):
    import torch
    rt = pkg.runtime
    with pytest.raises(rt.B2Error):
        rt.PagedKV.empty(4, 16, 2, 64, device="cpu")
    k = torch.zeros(4, 2, 24, 64, dtype=torch.int8)
    s = torch.zeros(4, 2, 1)
    with pytest.raises(rt.B2Error, match="page_size"):
        rt.PagedKV(k, k, s, s)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(rt.B2Error):
        rt.KVRows(i, i[:2], i[:2, None], 3)
    with pytest.raises(rt.B2Error):
        rt.qk_norm_rope(None, None, 64)
    with pytest.raises(rt.B2Error):
        rt.qk_norm_rope(torch.zeros(2, 64), None, 64)


@pytest.mark.parametrize("n_rows,n_seq,cap,H,KVH", [(16384, 2, 1 << 17, 32, 32), (8192, 9, 1 << 18, 32, 32), (30000, 40, 1 << 18, 12, 12)])
def test_long_prompts_over_a_large_capacity_are_accepted(pkg, n_rows, n_seq, cap, H, KVH):
    """Only a few rows of a call can be short sequences' single tokens: the rest does not count as pieces of that kind.
    (Without a workspace the call stops before its launch: what it says then is that it needs one.)"""
    rt = pkg.runtime
    r = rows(rt, n_rows=n_rows, n_seq=n_seq, max_pages=cap // 64)
    kv = pages(rt, n_pages=1 << 14, page_size=64, n_kv_heads=KVH, d_head=128)
    assert attend(rt, kv, r, n_heads=H, ldq=H * 128, ldo=H * 128, out=1 << 40, ws=None, ws_bytes=0) == -1
    assert "workspace" in rt.last_error()


@pytest.mark.parametrize("n_rows,n_seq,cap,H,KVH,dh,max_rows", [
    (8188, 4, 2047, 32, 8, 128, 2047), (2048, 9, 1 << 15, 32, 8, 128, 0), (8192, 9, 1 << 17, 32, 8, 128, 0), (8192, 9, 1 << 17, 32, 32, 256, 0),
    (5000, 3, 1 << 17, 64, 2, 64, 0), (40, 1, 1 << 20, 4, 1, 128, 0), (1, 1, 1 << 20, 128, 1, 256, 0), (100, 64, 1 << 15, 32, 8, 128, 0)])
def test_workspace_holds_the_rows_that_have_splits(pkg, n_rows, n_seq, cap, H, KVH, dh, max_rows):
    """Rows of short sequences (up to 16 columns of a KV head) in splits of 512 keys, and of the others as many as fill
    the GPU a few times (118 MB): not every row of the call in the finer splits."""
    rt = pkg.runtime
    r = rows(rt, n_rows=n_rows, n_seq=n_seq, max_pages=-(-cap // 64), max_keys=cap, max_rows=max_rows)
    kv = pages(rt, n_pages=1 << 14, page_size=64, n_kv_heads=KVH, d_head=dh)
    got = rt.lib().b2_attn_paged_i8_workspace(C.addressof(kv), C.addressof(r), H)
    short = min(n_rows, n_seq * (16 // (H // KVH))) if n_seq > 1 else 0
    assert got % 16 == 0 and got <= short * H * -(-cap // 512) * (dh + 4) * 4 + 118_000_000


def test_a_few_rows_of_many_slots_are_accepted(pkg):
    """Seventeen single tokens of 16384 slots over a large capacity: sequences without rows are no pieces."""
    rt = pkg.runtime
    r = rows(rt, n_rows=17, n_seq=16384, max_pages=(1 << 20) // 64)
    kv = pages(rt, n_pages=1 << 14, page_size=64, n_kv_heads=32, d_head=128)
    assert attend(rt, kv, r, n_heads=32, ldq=4096, ldo=4096, ws=None, ws_bytes=0) == -1
    assert "workspace" in rt.last_error()


def test_every_device_error_has_a_name_and_a_text(pkg):
    """The codes that the paged kernels set (paged.cuh) are named with the same values in the header, and check() has a
    text for each."""
    import re
    csrc = ROOT / "aricode-ml_b200" / "csrc"
    code = dict(re.findall(r"(B2_DEV_ERR_\w+) = (\d+)", (csrc / "b2_common.cuh").read_text()))
    used = {int(code[n]) for n in re.findall(r"set_err\([^;]*?(B2_DEV_ERR_\w+)\)", (csrc / "paged.cuh").read_text())}
    named = {int(v) for v in re.findall(r"B2_ROWS_\w+ = (\d+)", (ROOT / "include" / "b2dec.h").read_text())}
    assert used == named == set(pkg.runtime.ROWS_ERRORS) and len(used) >= 4


def test_read_only_loads_are_of_constants_alone():
    """The paged kernels start while the launch before them runs, and read-only loads want data that nothing writes in a
    kernel's lifetime: only gains and rotation tables are read that way, not what a launch may have written."""
    import re
    src = (ROOT / "aricode-ml_b200" / "csrc" / "paged.cuh").read_text().replace("(__ldg)", "")
    loads = [src[m.end():m.end() + 60] for m in re.finditer(r"__ldg\(", src)]
    assert loads
    for arg in loads:
        assert re.match(r"reinterpret_cast<const float4\*>\((p\.table|p\.nr\.table|p\.nr\.gk|g) \+", arg), arg


def test_more_sequences_than_a_call_can_search_are_refused(pkg):
    """A call's time grows with the square of its sequences: 0.4 s at the limit, minutes at a million."""
    rt = pkg.runtime
    for n_seq in (65537, 1 << 20):
        for call in (append, read, attend):
            assert call(rt, pages(rt), rows(rt, n_seq=n_seq)) == -1 and "65536" in rt.last_error()
    assert attend(rt, pages(rt), rows(rt, n_seq=65536, n_rows=200, max_pages=100), ws=None, ws_bytes=0) == -1
    assert "workspace" in rt.last_error()


def test_outputs_that_overlap_inputs_are_refused(pkg):
    """In place with the input's own stride, or beside it in one buffer, is fine (that is tested on the GPU); anything
    else would be read while it is written. Rows: 5 of 256 floats (q) and 128 (k, v), 1024 and 512 bytes."""
    rt = pkg.runtime
    far = A + (1 << 16)
    apart = dict(q=A, qo=A + 1 * far, k=A + 2 * far, ko=A + 3 * far, n_rows=5)
    for bad in (dict(qo=A, ldqo=512), dict(qo=A + 64), dict(qo=A + 4 * 1024 + 512), dict(qo=A - 4 * 1024), dict(ko=A + 2 * far, ldko=256),
                dict(qo=A + 2 * far), dict(ko=A), dict(ko=A + far + 512), dict(q=A, ldq=512, qo=A + 512, ldqo=512)):
        assert norm_rope(rt, **{**apart, **bad}) == -1 and "overlap" in rt.last_error(), bad
    kv, r = pages(rt), rows(rt)
    q = dict(q=far, ldq=256, q_out=2 * far, ldqo=256, n_heads=4, v=3 * far)
    for bad in (dict(q_out=far, ldqo=512), dict(q_out=far + 1024), dict(q_out=A), dict(q_out=3 * far + 16), dict(q_out=A - 4 * 1024)):
        assert append(rt, kv, r, **{**q, **bad}) == -1 and "overlap" in rt.last_error(), bad
    for bad in (dict(v=A), dict(v=A + 16), dict(v=A + 512 * 4), dict(bf16=1, v=A + 256 * 4), dict(ld=256, v=A + 256)):
        assert read(rt, kv, r, **bad) == -1 and "overlap" in rt.last_error(), bad
    for bad in (dict(out=A), dict(out=A + 1024), dict(out=A, ldo=512), dict(out=A + 256, ldo=256), dict(out=A - 4 * 1024),
                dict(ldq=512, ldo=512, out=A + 512)):
        assert attend(rt, kv, r, **bad) == -1 and "overlap" in rt.last_error(), bad
    # beside each other in one buffer: refused for the missing workspace alone
    for good in (dict(ldq=512, ldo=512, out=A + 1024), dict(ldq=1024, ldo=1024, out=A - 2048), dict(out=A + 5 * 1024)):
        assert attend(rt, kv, rows(rt, max_pages=5000), **good, ws=None) == -1 and "workspace" in rt.last_error(), good
