"""The paged 8-bit KV cache (qk_norm_rope, kv_append_i8, kv_read_i8, attn_paged_i8) against plain implementations in
64 bits.

Tolerances. u = 2^-24 is half a step of f32. A rounding model of independent errors is used: a sum of n terms is off
by at most 6 sqrt(n) u of its terms' magnitudes (six standard deviations), a handful of single operations by that many u.
What the cache holds is exact: a code times its scale is compared with an exact restatement in f32 where no sum comes
before it (values; keys without a norm), and else within half a code step."""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch


@pytest.fixture
def rt(pkg):
    return pkg.runtime


# ------------------------------------------------------------------ plain implementations
def turn64(torch, x, gain, table):
    """(result, magnitude): x [n, heads, d] in 64 bits normed by gain, its neighbouring pairs turned by table [n, d];
    the magnitude bounds what f32 roundings are relative to."""
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.double()
    if table is None:
        return x, x.abs()
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = table.double()[:, None, 0::2], table.double()[:, None, 1::2]
    y, m = torch.empty_like(x), torch.empty_like(x)
    y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    m[..., 0::2], m[..., 1::2] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, m


def turn_tol(mag, d):
    # sum of squares 6 sqrt(d) u (half of it through the root), mean, eps, root, divide, two products, rotation (2), scale
    return mag * (3 * math.sqrt(d) + 10) * U


def table64(torch, n, d):
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    return torch.stack((ang.cos(), ang.sin()), -1).reshape(n, d).float()


def pool(torch, rt, rows, keys, KVH, dh, page, seed=0, spare=2, extra_pages=1):
    """A cache holding random keys for sequences of `keys` tokens, in scattered pages; every scale that no key uses is
    NaN and every table entry past the keys is nonsense. Returns (PagedKV, KVRows arguments)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-k // page) for k in keys]
    n_pages, most = sum(need) + spare, max(need) + extra_pages
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(keys), most), -12345, dtype=torch.int32, device="cuda")
    kv = rt.PagedKV.empty(n_pages, page, KVH, dh)
    at = 0
    for s, (n, k) in enumerate(zip(need, keys)):
        table[s, :n] = order[at:at + n]
        at += n
    for name in ("k", "v"):
        codes = torch.randint(-127, 128, kv.k.shape, device="cuda", generator=g, dtype=torch.int8)
        scale = torch.full_like(kv.k_scale, float("nan"))
        for s, k in enumerate(keys):
            for b in range(-(-k // 16)):
                p = int(table[s, b * 16 // page])
                scale[p, :, b * 16 % page // 16] = 0.005 + 0.02 * torch.rand(KVH, device="cuda", generator=g)
        getattr(kv, name).copy_(codes)
        getattr(kv, name + "_scale").copy_(scale)
    return kv, ragged(torch, rows, keys, table)


def ragged(torch, rows, keys, table, pad=0):
    start = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    return dict(row_start=start, kv_len=torch.tensor(keys, dtype=torch.int32, device="cuda"), page_table=table,
                n_rows=sum(rows) + pad)


def held(torch, kv, table, s, n):
    """(k, v) of the first n keys of sequence s in 64 bits, [n, kv_heads, d]; None pages give zeros."""
    out = []
    for x, sc in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        rows = []
        for j0 in range(0, n, kv.page_size):
            p = int(table[s, j0 // kv.page_size])
            if not 0 <= p < kv.n_pages:
                rows.append(torch.zeros(kv.page_size, kv.n_kv_heads, kv.d_head, dtype=torch.float64, device="cuda"))
                continue
            rows.append((x[p].double() * sc[p].double().repeat_interleave(16, 1)[..., None]).transpose(0, 1))
        out.append(torch.cat(rows)[:n] if rows else torch.zeros(0, kv.n_kv_heads, kv.d_head, dtype=torch.float64, device="cuda"))
    return out


def attend64(torch, kv, plan, rows, keys, q, H, capacity=None):
    """(out, tolerance) [n, H, d] in 64 bits."""
    G, d = H // kv.n_kv_heads, kv.d_head
    outs, tols, a = [], [], 0
    for s, (r, kn) in enumerate(zip(rows, keys)):
        n = min(kn, capacity or kn)
        k, v = held(torch, kv, plan["page_table"], s, n)
        vcode_top = kv.v_scale.nan_to_num(0.0).amax().double() * 127
        page = plan["page_table"][s, torch.arange(n, device="cuda") // kv.page_size]
        there = (page >= 0) & (page < kv.n_pages)
        qs = q[a:a + r].reshape(r, H, d).double()
        k, v = k.repeat_interleave(G, 1).transpose(0, 1), v.repeat_interleave(G, 1).transpose(0, 1)   # [H, n, d]
        pos = torch.arange(kn - r, kn, device="cuda")
        seen = (torch.arange(n, device="cuda")[None, :] <= pos[:, None]) & there[None, :]              # [r, n]
        score = (qs.transpose(0, 1) @ k.transpose(1, 2)).masked_fill(~seen, -math.inf)
        none = ~seen.any(1)
        p = torch.softmax(score, -1).nan_to_num(0.0) if n else score
        if n:
            p = torch.where(none[None, :, None], 0.0, torch.softmax(score.masked_fill(none[None, :, None], 0.0), -1))
        out = p @ v
        # scores: the sum over d, and queries held to 2^-23 of their head's largest; exponentials: the argument's
        # rounding and a few u; sums over the keys; weights held to 2^-23 of the largest of their neighbours
        mag = (qs.abs().transpose(0, 1) @ k.abs().transpose(1, 2)).masked_fill(~seen, 0.0)
        top = qs.abs().amax(-1).T[:, :, None] * k.square().sum(-1).sqrt()[:, None, :]
        e_s = ((6 * math.sqrt(d) + 8) * mag + 6 * top.masked_fill(~seen, 0.0)).amax(-1, keepdim=True) * U if n else 0.0
        spread = (score.masked_fill(~seen, -math.inf).amax(-1, keepdim=True) - score.masked_fill(~seen, math.inf).amin(-1, keepdim=True)).clamp(0, 104).nan_to_num(0.0) if n else 0.0
        rel = 2 * e_s + (2 * spread + 16 + 12 * math.sqrt(max(n, 1))) * U
        tol = rel * (p @ v.abs()) + 6 * math.sqrt(max(n, 1)) * U * vcode_top * (p.amax(-1, keepdim=True) if n else 0.0)
        outs.append(out.transpose(0, 1))
        tols.append(tol.transpose(0, 1))
        a += r
    return torch.cat(outs), torch.cat(tols)


def close(torch, got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= tol)                                            # a NaN is bad
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(off[bad].max())} against {float(tol[bad].max())}"


# ------------------------------------------------------------------ norm and rotation
@pytest.mark.parametrize("n,H,KVH,dh", [(1, 32, 4, 64), (3, 4, 2, 16), (7, 5, 3, 48), (33, 32, 8, 128), (2, 3, 1, 256),
                                        (5, 7, 7, 80), (600, 12, 12, 144), (1500, 32, 8, 128)])
@pytest.mark.parametrize("which", ["both", "norm", "rope", "scale"])
def test_norm_rope(torch, rt, n, H, KVH, dh, which):
    g = torch.Generator(device="cuda").manual_seed(n * 7 + dh)
    qkv = torch.randn(n, (H + 2 * KVH) * dh + 4, device="cuda", generator=g) * 3
    q, k = qkv[:, :H * dh], qkv[:, H * dh:(H + KVH) * dh]
    gq, gk = (1 + torch.randn(2, dh, device="cuda", generator=g)) if which in ("both", "norm") else (None, None)
    table = table64(torch, 97, dh) if which in ("both", "rope") else None
    pos = torch.randint(0, 97, (n,), device="cuda", generator=g).to(torch.int32) if table is not None else None
    qo, ko = rt.qk_norm_rope(q, k, dh, pos=pos, table=table, q_gain=gq, k_gain=gk, eps=EPS, q_scale=0.25)
    for x, gain, got, sc, heads in ((q, gq, qo, 0.25, H), (k, gk, ko, 1.0, KVH)):
        want, mag = turn64(torch, x.reshape(n, heads, dh), gain, None if table is None else table[pos.long()])
        close(torch, got.reshape(n, heads, dh), want * sc, turn_tol(mag * sc, dh) + 1e-45)


def test_norm_rope_in_place_one_gain_padding_and_range(torch, rt):
    """In place on strided rows; a gain for the keys alone; rows with pos < 0 and rows past the table are left as they
    were, and only the latter set the error word."""
    n, H, KVH, dh = 9, 4, 2, 64
    buf = torch.randn(n, (H + KVH) * dh + 8, device="cuda")
    q, k = buf[:, :H * dh], buf[:, H * dh:(H + KVH) * dh]
    before, table, gk = buf.clone(), table64(torch, 5, dh), torch.rand(dh, device="cuda")
    pos = torch.tensor([0, -1, 4, 3, 5, 2 ** 31 - 1, -2 ** 31, 1, 2], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rt.qk_norm_rope(q, k, dh, pos=pos, table=table, k_gain=gk, eps=EPS, q_out=q, k_out=k, err=err)
    ok = (pos >= 0) & (pos < 5)
    assert torch.equal(buf[~ok], before[~ok]) and torch.equal(buf[:, (H + KVH) * dh:], before[:, (H + KVH) * dh:])
    assert int(err) == 2
    for x, got, gain, heads in ((before[:, :H * dh], q, None, H), (before[:, H * dh:(H + KVH) * dh], k, gk, KVH)):
        want, mag = turn64(torch, x[ok].reshape(-1, heads, dh), gain, table[pos[ok].long()])
        close(torch, got[ok].reshape(-1, heads, dh), want, turn_tol(mag, dh))


def test_norm_rope_equals_rope_apply_bit_for_bit(torch, rt):
    x = torch.randn(1, 3 * 64, device="cuda")
    table = table64(torch, 40, 64)
    a, _ = rt.qk_norm_rope(x, None, 64, pos=torch.tensor([37], dtype=torch.int32, device="cuda"), table=table)
    assert torch.equal(a[0], rt.rope_apply(x[0].clone(), table, 37, 64))


# ------------------------------------------------------------------ append and read
def quantise(torch, codes, scale, rows, o0):
    """One block of one head in f32, as documented: codes [16, d] int8, scale a 0-d f32, rows [n, d] f32 written at
    o0. Returns the new (codes, scale)."""
    codes, old = codes.clone(), torch.zeros_like(scale) if o0 == 0 else scale
    top = rows.abs().max()
    # by a tensor: a division by a number is a product with its reciprocal in torch
    now = torch.where(torch.isfinite(rows).all(), top / torch.full_like(top, 127.0), torch.full_like(top, float("nan")))
    now = torch.where(torch.isnan(old) | torch.isnan(now), torch.full_like(top, float("nan")), torch.maximum(old, now))
    if o0 and bool(now > old):
        codes[:o0] = (codes[:o0].float() * (old / now)).round().to(torch.int8)
    new = (rows / now).round().clamp(-127, 127) if bool(now > 0) else torch.zeros_like(rows)
    codes[o0:o0 + rows.shape[0]] = new.to(torch.int8)
    return codes, now


def append_plain(torch, kv, plan, rows, keys, x, name, capacity=10 ** 9):
    """What kv_append_i8 leaves in k or v for f32 rows x [n, kv_heads, d] written as they are."""
    codes, scale = getattr(kv, name).clone(), getattr(kv, name + "_scale").clone()
    a = 0
    for s, (r, kn) in enumerate(zip(rows, keys)):
        first = max(kn - r, 0)
        for b in range(first // 16 * 16, min(kn, capacity), 16):
            lo, hi = max(b, first), min(b + 16, kn, capacity)
            if lo >= hi:
                continue
            p, blk = int(plan["page_table"][s, b // kv.page_size]), b % kv.page_size // 16
            if not 0 <= p < kv.n_pages:
                continue
            for h in range(kv.n_kv_heads):
                part = x[a + lo - (kn - r):a + hi - (kn - r), h]
                cell = codes[p, h, blk * 16:blk * 16 + 16]
                codes[p, h, blk * 16:blk * 16 + 16], scale[p, h, blk] = quantise(torch, cell, scale[p, h, blk], part, lo - b)
        a += r
    return codes, scale


def same_cache(torch, kv, want):
    for name, (codes, scale) in want.items():
        got = getattr(kv, name + "_scale")
        assert torch.equal(got.view(torch.int32).where(~got.isnan(), 0), scale.view(torch.int32).where(~scale.isnan(), 0))
        assert torch.equal(got.isnan(), scale.isnan())
        assert torch.equal(getattr(kv, name), codes)


CASES = [([1], [1]), ([1], [16]), ([1], [17]), ([1, 1, 1], [40, 16, 33]), ([5, 0, 20, 1], [5, 9, 35, 64]), ([40], [40]),
         ([37, 50], [64, 70]), ([6], [2]), ([0, 0], [3, 0]), ([130, 3], [200, 3])]


@pytest.mark.parametrize("rows,keys", CASES)
@pytest.mark.parametrize("KVH,dh,page", [(2, 64, 16), (3, 128, 32), (1, 16, 64), (2, 80, 16), (5, 32, 128), (1, 256, 32)])
def test_append_and_read_are_exact(torch, rt, rows, keys, KVH, dh, page):
    """Without norm or rotation the codes and scales are those of the documented f32 arithmetic, bit for bit; nothing
    else in the pool changes; reading back gives code times scale."""
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page, seed=len(rows))
    n = sum(rows)
    x = [torch.randn(n + 2, KVH * dh, device="cuda") * (0.2 + 3 * torch.rand(n + 2, 1, device="cuda")) for _ in range(2)]
    want = {name: append_plain(torch, kv, plan, rows, keys, y.reshape(n + 2, KVH, dh), name) for name, y in zip("kv", x)}
    r = rt.KVRows(**{**plan, "n_rows": n + 2})
    rt.kv_append_i8(kv, r, x[0], x[1])
    same_cache(torch, kv, want)
    kv.check()
    for dtype in (torch.float32, torch.bfloat16):
        outs = [torch.full((n + 2, KVH * dh), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        got = rt.kv_read_i8(kv, r, k_out=outs[0], v_out=outs[1])
        a = 0
        for s, (rr, kn) in enumerate(zip(rows, keys)):
            first = max(kn - rr, 0)
            skip = rr - (kn - first)                               # rows before position 0
            for y, h in zip(got, held(torch, kv, plan["page_table"], s, kn)):
                assert torch.equal(y[a + skip:a + rr].double(), h[first:kn].reshape(-1, KVH * dh).float().to(dtype).double())
                assert bool((y[a:a + skip] == 7).all())
            a += rr
        assert bool((got[0][n:] == 7).all()) and bool((got[1][n:] == 7).all())


@pytest.mark.parametrize("H,KVH,dh,page", [(8, 2, 128, 16), (6, 3, 64, 64), (4, 2, 16, 16), (2, 2, 192, 32)])
@pytest.mark.parametrize("rows,keys", [([1, 1], [9, 33]), ([20, 0, 45], [20, 5, 90])])
def test_append_norms_and_rotates_on_the_way(torch, rt, H, KVH, dh, page, rows, keys):
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page, seed=3)
    n, first_held = sum(rows), [held(torch, kv, plan["page_table"], s, k) for s, k in enumerate(keys)]
    g = torch.Generator(device="cuda").manual_seed(11)
    qkv = torch.randn(n, (H + 2 * KVH) * dh, device="cuda", generator=g)
    q, k, v = qkv[:, :H * dh], qkv[:, H * dh:(H + KVH) * dh], qkv[:, (H + KVH) * dh:]
    gq, gk = 1 + 0.3 * torch.randn(2, dh, device="cuda", generator=g)
    table = table64(torch, 128, dh)
    r = rt.KVRows(**plan)
    pos = torch.cat([torch.arange(kn - rr, kn, device="cuda") for rr, kn in zip(rows, keys)]).to(torch.int32)
    qo = rt.kv_append_i8(kv, r, k, v, table=table, k_gain=gk, eps=EPS, q=q, q_gain=gq, q_scale=0.5)
    q2, _ = rt.qk_norm_rope(q, k, dh, pos=pos, table=table, q_gain=gq, k_gain=gk, eps=EPS, q_scale=0.5)
    assert torch.equal(qo, q2)                                     # one arithmetic in both calls
    want, mag = turn64(torch, k.reshape(n, KVH, dh), gk, table[pos.long()])
    tol = turn_tol(mag, dh)
    a = 0
    for s, (rr, kn) in enumerate(zip(rows, keys)):
        got = held(torch, kv, plan["page_table"], s, kn)[0]
        for b in range((kn - rr) // 16 * 16, kn, 16):
            lo, hi = max(b, kn - rr), min(b + 16, kn)
            if lo >= hi:
                continue
            part, pt = want[a + lo - (kn - rr):a + hi - (kn - rr)], tol[a + lo - (kn - rr):a + hi - (kn - rr)]
            p, blk = int(plan["page_table"][s, b // page]), b % page // 16
            scale = kv.k_scale[p, :, blk].double()
            top = part.abs().amax((0, 2)) / 127
            if lo > b:
                top = torch.maximum(top, first_held[s][0][b:lo].abs().amax((0, 2)) / 127)   # at least what is there needs
            assert bool((scale >= top * (1 - 1e-5)).all())
            # half a step, and what f32 did before the code was chosen
            close(torch, got[lo:hi], part, 0.5 * scale[None, :, None] * (1 + 1e-5) + pt)
            if lo > b:                                             # older rows moved by at most half a step of the new scale
                close(torch, got[b:lo], first_held[s][0][b:lo], (0.5 * scale[None, :, None] * (1 + 1e-5)).expand(lo - b, -1, dh))
        a += rr
    kv.check()


def test_tokens_one_by_one_keep_their_values(torch, rt):
    """Sixteen tokens of growing size appended singly: the block's scale ends where one call puts it, and each value is
    within half a step of every scale it went through."""
    KVH, dh = 2, 64
    x = torch.randn(16, KVH * dh, device="cuda") * torch.linspace(0.1, 4, 16, device="cuda")[:, None]
    kv = rt.PagedKV.empty(2, 16, KVH, dh)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    steps = torch.zeros(KVH, dtype=torch.float64, device="cuda")
    bound = torch.zeros(16, KVH, dtype=torch.float64, device="cuda")
    for i in range(16):
        rt.kv_append_i8(kv, rt.KVRows(**ragged(torch, [1], [i + 1], table)), x[i:i + 1], x[i:i + 1])
        now = kv.k_scale[1, :, 0].double()
        bound[:i] += torch.where(now > steps, 0.5 * now * (1 + 1e-5), 0.0)
        bound[i] = 0.5 * now * (1 + 1e-5)
        steps = now
    one = rt.PagedKV.empty(2, 16, KVH, dh)
    rt.kv_append_i8(one, rt.KVRows(**ragged(torch, [16], [16], table)), x, x)
    assert torch.equal(one.k_scale, kv.k_scale) and torch.equal(one.v_scale, kv.v_scale)
    close(torch, held(torch, kv, table, 0, 16)[0], x.reshape(16, KVH, dh).double(), bound[..., None].expand(-1, -1, dh))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_append_of_a_non_finite_value(torch, rt, value):
    """Its block's scale becomes NaN (of that head, keys or values alone), stays so while the block grows, and is fresh
    when the block is written from its start again."""
    kv = rt.PagedKV.empty(3, 16, 2, 32)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 64, device="cuda")
    y = x.clone()
    y[3, 40] = value
    rt.kv_append_i8(kv, rt.KVRows(**ragged(torch, [4], [4], table)), y, x)
    assert bool(kv.k_scale[2, 1, 0].isnan()) and int(kv.k_scale.isnan().sum()) == 1 and not bool(kv.v_scale.isnan().any())
    rt.kv_append_i8(kv, rt.KVRows(**ragged(torch, [1], [5], table)), x[:1], x[:1])
    assert bool(kv.k_scale[2, 1, 0].isnan())
    out = rt.attn_paged_i8(kv, rt.KVRows(**ragged(torch, [1], [5], table)), torch.randn(1, 64, device="cuda"))
    assert bool(out[0, 32:].isnan().all()) and bool(out[0, :32].isfinite().all())
    rt.kv_append_i8(kv, rt.KVRows(**ragged(torch, [4], [4], table)), x, x)
    assert bool(kv.k_scale.isfinite().all())


def test_append_of_zeros_and_tiny_values(torch, rt):
    kv = rt.PagedKV.empty(1, 16, 1, 16)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 16, device="cuda")
    x[1] = torch.linspace(-1, 1, 16, device="cuda") * 3e-44         # a few steps of the smallest f32: a scale of 0
    r = rt.KVRows(**ragged(torch, [2], [2], table))
    rt.kv_append_i8(kv, r, torch.zeros_like(x), x)
    assert float(kv.k_scale[0, 0, 0]) == 0.0 and int(kv.k.abs().sum()) == 0
    want = append_plain(torch, rt.PagedKV.empty(1, 16, 1, 16), ragged(torch, [2], [2], table), [2], [2], x.reshape(2, 1, 16), "v")
    assert torch.equal(kv.v_scale, want[1]) and torch.equal(kv.v, want[0])
    assert bool((rt.attn_paged_i8(kv, r, torch.ones(2, 16, device="cuda")) == 0).all()) or float(kv.v_scale.max()) > 0


def test_bad_pages_and_lengths_are_left_out(torch, rt):
    """Entries outside the pool, keys past the capacity and rows past the table: left out, with the error word set."""
    rows, keys, KVH, dh, page = [20, 3], [40, 35], 2, 64, 16
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page)
    x = torch.randn(23, KVH * dh, device="cuda")
    for entry in (-1, kv.n_pages, 2 ** 31 - 1, -2 ** 31):
        plan["page_table"][0, 1] = entry                           # positions 16 to 31 of sequence 0
        want = {n: append_plain(torch, kv, plan, rows, keys, x.reshape(23, KVH, dh), n) for n in "kv"}
        r = rt.KVRows(**plan)
        rt.kv_append_i8(kv, r, x, x)
        same_cache(torch, kv, want)
        with pytest.raises(rt.B2Error, match="page-table entry"):
            kv.check()
        got = rt.kv_read_i8(kv, r)[0]
        assert bool((got[:12] == 0).all()) and not bool((got[12:20] == 0).all())
        with pytest.raises(rt.B2Error):
            kv.check()
        kv.check()                                                 # cleared
        q = torch.randn(23, 4 * dh, device="cuda") * 0.2
        out = rt.attn_paged_i8(kv, r, q)
        close(torch, out.reshape(23, 4, dh), *attend64(torch, kv, plan, rows, keys, q, 4))
        with pytest.raises(rt.B2Error, match="page-table entry"):
            kv.check()
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page)
    want = {n: append_plain(torch, kv, plan, rows, keys, x.reshape(23, KVH, dh), n, capacity=37) for n in "kv"}
    r = rt.KVRows(**plan, max_keys=37)
    rt.kv_append_i8(kv, r, x, x)
    same_cache(torch, kv, want)
    with pytest.raises(rt.B2Error, match="capacity"):
        kv.check()
    out = rt.attn_paged_i8(kv, r, q)
    close(torch, out.reshape(23, 4, dh), *attend64(torch, kv, plan, rows, keys, q, 4, capacity=37))
    with pytest.raises(rt.B2Error, match="capacity"):
        kv.check()
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page)
    want = {n: append_plain(torch, kv, plan, rows, keys, x.reshape(23, KVH, dh), n, capacity=36) for n in "v"}
    rt.kv_append_i8(kv, rt.KVRows(**plan), x, x, table=table64(torch, 36, dh))
    same_cache(torch, kv, want)
    with pytest.raises(rt.B2Error, match="table"):
        kv.check()


def test_odd_row_ranges(torch, rt):
    """Starts that go down, point outside or are negative, and lengths that are: nothing outside the buffers is
    touched, and rows of no sequence keep their outputs."""
    kv, plan = pool(torch, rt, [4, 4, 4], [10, 20, 30], 1, 32, 16)
    x = torch.randn(12, 32, device="cuda")
    for start, lens in (([0, 4, 2, 12], [10, 20, 30]), ([-5, 4, 8, 900], [10, 20, 30]), ([3, 3, 3, 3], [1, 2, 3]),
                        ([0, 4, 8, 12], [-7, -2 ** 31, 30]), ([0, 12, 0, 12], [30, 20, 30])):
        p = dict(plan, row_start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                 kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        r = rt.KVRows(**p)
        rt.kv_append_i8(kv, r, x, x)
        out = torch.full((14, 64), 5.0, device="cuda")
        rt.attn_paged_i8(kv, r, torch.randn(14, 64, device="cuda"), out=out)
        rt.kv_read_i8(kv, r)
        torch.cuda.synchronize()
        assert bool((out[12:] == 5).all())
        if start == [3, 3, 3, 3]:
            assert bool((out == 5).all())
        kv.err.zero_()


# ------------------------------------------------------------------ attention
HEADS = [(32, 32, 128, 16), (32, 4, 64, 32), (4, 2, 16, 16), (8, 1, 80, 64), (6, 6, 256, 16), (14, 7, 96, 128),
         (48, 2, 32, 16), (40, 1, 128, 1024), (12, 12, 64, 16), (6, 2, 192, 32)]
LENGTHS = [([1], [1]), ([1], [640]), ([1, 1, 0, 1], [1, 17, 5, 300]), ([5, 0, 33, 1], [5, 9, 40, 64]), ([6], [2]),
           ([2, 9], [700, 130]), ([64, 65], [64, 65]), ([130], [513]), ([0, 1], [0, 257])]


@pytest.mark.parametrize("H,KVH,dh,page", HEADS)
@pytest.mark.parametrize("rows,keys", LENGTHS)
def test_attention(torch, rt, H, KVH, dh, page, rows, keys):
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page, seed=dh)
    n = sum(rows)
    g = torch.Generator(device="cuda").manual_seed(n)
    # strided rows, some heads sharp
    q = torch.randn(n + 3, H * dh + 8, device="cuda", generator=g)[:, :H * dh]
    q *= (dh ** -0.5 * (0.3 + 3 * torch.rand(H, device="cuda", generator=g))).repeat_interleave(dh)
    out = torch.full((n + 3, H * dh + 4), 9.0, device="cuda")
    rt.attn_paged_i8(kv, rt.KVRows(**{**plan, "n_rows": n + 3}, max_rows=max(rows)), q, out=out[:, :H * dh])
    want, tol = attend64(torch, kv, plan, rows, keys, q, H)
    close(torch, out[:n, :H * dh].reshape(n, H, dh), want, tol)
    assert bool((out[n:] == 9).all()) and bool((out[:, H * dh:] == 9).all())
    kv.check()
    # without the hints: the same sequences
    again = rt.attn_paged_i8(kv, rt.KVRows(**plan), q)
    close(torch, again[:n].reshape(n, H, dh), want, tol)


@pytest.mark.parametrize("H,KVH,dh,page,rows,keys", [
    (32, 8, 128, 64, [1] * 40, list(range(1, 4000, 100))), (32, 32, 128, 64, [1], [9000]), (8, 1, 64, 256, [1, 1], [40001, 33]),
    (16, 2, 128, 16, [300, 1, 77], [300, 5000, 2100]), (4, 4, 128, 32, [1030], [1030]), (8, 8, 64, 16, [3], [20000])])
def test_attention_long(torch, rt, H, KVH, dh, page, rows, keys):
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, page, seed=2)
    n = sum(rows)
    q = torch.randn(n, H * dh, device="cuda") * 1.5 * dh ** -0.5
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan, max_keys=max(keys), max_rows=max(rows)), q)
    close(torch, out.reshape(n, H, dh), *attend64(torch, kv, plan, rows, keys, q, H))
    kv.check()


def test_attention_of_extreme_scores(torch, rt):
    """Scores in the hundreds (one key takes all), all equal scores (zero queries), and a query with one huge element."""
    rows, keys, H, KVH, dh = [3, 1], [90, 200], 4, 2, 64
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 16)
    for q in (torch.randn(4, H * dh, device="cuda") * 60, torch.zeros(4, H * dh, device="cuda"),
              torch.randn(4, H * dh, device="cuda") * torch.where(torch.arange(H * dh, device="cuda") % dh == 5, 50.0, 1e-3),
              torch.full((4, H * dh), 1e-38, device="cuda"), torch.full((4, H * dh), 1e-42, device="cuda")):
        out = rt.attn_paged_i8(kv, rt.KVRows(**plan), q)
        close(torch, out.reshape(4, H, dh), *attend64(torch, kv, plan, rows, keys, q, H))


def test_attention_of_non_finite_queries(torch, rt):
    """A NaN or infinity in one head's query: that head's row is NaN, no other."""
    kv, plan = pool(torch, rt, [2, 1], [50, 600], 2, 64, 16)
    q = torch.randn(3, 4 * 64, device="cuda") * 0.1
    q[0, 70], q[2, 3] = float("nan"), float("inf")
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan), q).reshape(3, 4, 64)
    bad = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[2, 0] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)


def test_attention_of_a_nan_block(torch, rt):
    """A key block whose scale is NaN makes the rows that see it NaN; a value block too; rows before it are finite."""
    for name in ("k_scale", "v_scale"):
        kv, plan = pool(torch, rt, [60], [60], 1, 64, 16)
        getattr(kv, name)[int(plan["page_table"][0, 2]), 0, 0] = float("nan")      # keys 32 to 47
        out = rt.attn_paged_i8(kv, rt.KVRows(**plan), torch.randn(60, 2 * 64, device="cuda") * 0.1)
        assert bool(out[:32].isfinite().all()) and bool(out[32:].isnan().all())


def test_a_pool_of_more_than_four_gib(torch, rt):
    """Offsets past 32 bits: the sequence's pages are the last of a 4.5 GB pool (K and V each)."""
    KVH, dh, page = 8, 128, 64
    n_pages = (9 << 29) // (KVH * dh * page)
    codes = [torch.empty(n_pages, KVH, page, dh, dtype=torch.int8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(n_pages, KVH, page // 16, device="cuda") for _ in range(2)]
    kv = rt.PagedKV(*codes, *scale)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2, n_pages - 3]], dtype=torch.int32, device="cuda")
    x = torch.randn(200, KVH * dh, device="cuda")
    plan = ragged(torch, [200], [200], table)
    want = x.reshape(200, KVH, dh).double()
    rt.kv_append_i8(kv, rt.KVRows(**plan), x, x)
    got = rt.kv_read_i8(kv, rt.KVRows(**plan))[1].reshape(200, KVH, dh)
    close(torch, got, want, want.abs().amax() / 127 * 0.5 * (1 + 1e-5) * torch.ones_like(want))
    q = torch.randn(200, 8 * dh, device="cuda") * dh ** -0.5
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan), q)
    close(torch, out.reshape(200, 8, dh), *attend64(torch, kv, plan, [200], [200], q, 8))


def test_rows_do_not_depend_on_the_other_sequences(torch, rt):
    """A sequence's single-token rows are the same bits alone and in a batch."""
    rows, keys, H, KVH, dh = [1] * 9, [700, 1, 64, 1300, 33, 256, 257, 16, 999], 16, 4, 128
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 16)
    q = torch.randn(9, H * dh, device="cuda") * dh ** -0.5
    both = rt.attn_paged_i8(kv, rt.KVRows(**plan, max_rows=1), q)
    for s in range(9):
        one = ragged(torch, [1], [keys[s]], plan["page_table"][s:s + 1].contiguous())
        assert torch.equal(rt.attn_paged_i8(kv, rt.KVRows(**one, max_rows=1), q[s:s + 1])[0], both[s])


@pytest.mark.parametrize("H,KVH,dh,rows,keys,cap", [
    (32, 8, 128, [40], [9000], 9000), (32, 8, 128, [40, 1, 64, 30], [300, 9000, 4097, 31], 20000), (12, 12, 64, [20] * 5, [2500, 20, 700, 4000, 1], 0),
    (16, 2, 80, [5, 3], [6000, 5999], 6000), (32, 8, 64, [17] + [1] * 260, [5000] + [40] * 260, 0), (8, 8, 128, [17, 0, 16], [0, 0, 3000], 0)])
def test_pieces_over_caches_of_very_different_lengths(torch, rt, H, KVH, dh, rows, keys, cap):
    """Pieces of prompts over caches of very different lengths, also far below the capacity; calls again are the same bits."""
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 32, seed=4)
    n = sum(rows)
    q = torch.randn(n, H * dh, device="cuda") * dh ** -0.5
    r = rt.KVRows(**plan, max_keys=cap)
    out = rt.attn_paged_i8(kv, r, q)
    close(torch, out.reshape(n, H, dh), *attend64(torch, kv, plan, rows, keys, q, H))
    kv.check()
    assert torch.equal(rt.attn_paged_i8(kv, r, q), out)


def test_prompts_beside_single_tokens(torch, rt):
    """A whole prompt beside single tokens with long caches: the prompt's rows have no splits to join, the tokens' have."""
    rows, keys, H, KVH, dh = [2000, 1, 3, 1], [2000, 3000, 700, 1], 32, 8, 128
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 64, seed=8)
    q = torch.randn(sum(rows), H * dh, device="cuda") * dh ** -0.5
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan, max_keys=3000), q)
    want, tol = attend64(torch, kv, plan, rows, keys, q, H)
    close(torch, out.reshape(-1, H, dh), want, tol)


def test_many_sequences(torch, rt):
    """600 sequences (the searches for a sequence go over 32 at a time), some without rows: append, read and attend."""
    n, H, KVH, dh = 600, 4, 2, 64
    keys = [(7 * s) % 90 + 1 for s in range(n)]
    rows = [0 if s % 11 == 3 else 1 if s % 5 else min(3, keys[s]) for s in range(n)]
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 32)
    r = rt.KVRows(**plan)
    T = sum(rows)
    x = torch.randn(T, KVH * dh, device="cuda")
    want = append_plain(torch, kv, plan, rows, keys, x.reshape(T, KVH, dh), "v")
    rt.kv_append_i8(kv, r, x, x)
    assert torch.equal(kv.v, want[0])
    got = rt.kv_read_i8(kv, r)[1].reshape(T, KVH, dh)
    a = 0
    for s in range(n):
        h = held(torch, kv, plan["page_table"], s, keys[s])[1]
        assert torch.equal(got[a:a + rows[s]].double(), h[keys[s] - rows[s]:].float().double())
        a += rows[s]
    q = torch.randn(T, H * dh, device="cuda") * 0.1
    close(torch, rt.attn_paged_i8(kv, r, q).reshape(T, H, dh), *attend64(torch, kv, plan, rows, keys, q, H))
    kv.check()


def test_hints_that_are_wrong_and_an_empty_table(torch, rt):
    """max_rows below the truth costs time, not results; without pages nothing is seen or written."""
    rows, keys, H, KVH, dh = [40, 1], [60, 500], 8, 2, 64
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 16)
    q = torch.randn(41, H * dh, device="cuda") * 0.1
    want, tol = attend64(torch, kv, plan, rows, keys, q, H)
    for hint in (1, 3, 41, 4000):
        close(torch, rt.attn_paged_i8(kv, rt.KVRows(**plan, max_rows=hint), q).reshape(41, H, dh), want, tol)
    kv.check()
    empty = dict(plan, page_table=torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    before = kv.k.clone()
    r = rt.KVRows(**empty)
    x = torch.randn(41, KVH * dh, device="cuda")
    rt.kv_append_i8(kv, r, x, x)
    assert torch.equal(kv.k, before) and bool((rt.attn_paged_i8(kv, r, q) == 0).all())
    with pytest.raises(rt.B2Error, match="capacity"):
        kv.check()


# ------------------------------------------------------------------ together
def test_a_layer_decoded_step_by_step(torch, rt):
    """Prompts of three sequences, then tokens: append (norm, rotation, queries on the way) and attend, each step
    against attention in 64 bits over the values that the cache then holds, and the whole against the values that went in."""
    H, KVH, dh, page, lens = 8, 2, 64, 16, [30, 1, 47]
    table = torch.randperm(3 * 8, device="cuda").to(torch.int32).reshape(3, 8)
    kv = rt.PagedKV.empty(24, page, KVH, dh)
    tab = table64(torch, 128, dh)
    gq, gk = 1 + 0.2 * torch.randn(2, dh, device="cuda")
    held_now, all_v = [0, 0, 0], [[] for _ in lens]
    for step in range(12):
        rows = lens if step == 0 else [1, 0 if step == 5 else 1, 1]
        held_now = [a + b for a, b in zip(held_now, rows)]
        plan = ragged(torch, rows, held_now, table)
        n = sum(rows)
        qkv = torch.randn(n, (H + 2 * KVH) * dh, device="cuda")
        q, k, v = qkv[:, :H * dh], qkv[:, H * dh:(H + KVH) * dh], qkv[:, (H + KVH) * dh:]
        r = rt.KVRows(**plan)
        qo = rt.kv_append_i8(kv, r, k, v, table=tab, k_gain=gk, eps=EPS, q=q, q_gain=gq, q_scale=dh ** -0.5)
        out = rt.attn_paged_i8(kv, r, qo)
        close(torch, out.reshape(n, H, dh), *attend64(torch, kv, plan, rows, held_now, qo, H))
        a = 0
        for s, rr in enumerate(rows):
            all_v[s].append(v[a:a + rr])
            a += rr
    kv.check()
    for s in range(3):
        v = torch.cat(all_v[s]).reshape(-1, KVH, dh).double()
        got = held(torch, kv, table, s, held_now[s])[1]
        # at most 15 moves of the scale, each within half a step of the last one
        step = torch.cat([kv.v_scale[int(table[s, b]), :, 0].double()[None].expand(16, -1) for b in range(8)])[:held_now[s]]
        close(torch, got, v, (8 * step)[..., None].expand_as(v))


def test_against_the_f32_cache_attention(torch, rt):
    """On the values of kv_read_i8 the framework's f32 decode attention agrees (its -60 tail weighs nothing here)."""
    H, KVH, dh, n = 8, 4, 128, 333
    kv, plan = pool(torch, rt, [1], [n], KVH, dh, 32)
    whole = rt.KVRows(**ragged(torch, [n], [n], plan["page_table"]))
    k, v = rt.kv_read_i8(kv, whole)
    q = torch.randn(1, H * dh, device="cuda") * dh ** -0.5
    ref = rt.attn_decode(q[0], *(x.reshape(n, KVH, dh).transpose(0, 1).contiguous() for x in (k, v)), H, KVH, dh, n, n)
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan), q)
    _, tol = attend64(torch, kv, plan, [1], [n], q, H)
    close(torch, out.reshape(H, dh), ref.reshape(H, dh).double(), 2 * tol[0])


def test_captured_step_replays_with_new_lengths(torch, rt):
    """Append and attend captured once; lengths, rows and inputs change in place between replays."""
    H, KVH, dh, page = 8, 2, 128, 16
    table = torch.randperm(2 * 40, device="cuda").to(torch.int32).reshape(2, 40)
    kv, eager = (rt.PagedKV.empty(80, page, KVH, dh) for _ in range(2))
    plan = ragged(torch, [1, 1], [1, 1], table)
    rows = rt.KVRows(**plan, max_rows=1)
    q, k, v = (torch.zeros(2, w * dh, device="cuda") for w in (H, KVH, KVH))
    out, qo = torch.zeros(2, H * dh, device="cuda"), torch.zeros(2, H * dh, device="cuda")
    tab = table64(torch, 640, dh)
    ws = rt.attn_paged_workspace(kv, rows, H)

    def step(c):
        rt.kv_append_i8(c, rows, k, v, table=tab, q=q, q_scale=dh ** -0.5, q_out=qo)
        rt.attn_paged_i8(c, rows, qo, out=out, workspace=ws)

    step(kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kv)
    for c in (kv.k, kv.v, kv.k_scale, kv.v_scale):
        c.zero_()
    lens = [0, 0]
    for i in range(60):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        live = [1, i % 3 != 1]
        add = 9 if i % 7 == 3 else 1                               # positions may also jump (the rows between are as they are)
        lens = [lens[0] + add, lens[1] + int(live[1])]
        plan["row_start"].copy_(torch.tensor([0, 1, 1 + int(live[1])], dtype=torch.int32))
        plan["kv_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        step(eager)
        assert torch.equal(got[:1 + int(live[1])], out[:1 + int(live[1])]), i
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(kv, name), getattr(eager, name))


def test_streams_and_reused_memory(torch, rt):
    """Calls given a stream of their own: the outputs that they make belong to it, and nothing runs on another."""
    kv, plan = pool(torch, rt, [1] * 4, [900, 30, 2000, 1], 4, 128, 16)
    r = rt.KVRows(**plan, max_rows=1)
    q = torch.randn(4, 8 * 128, device="cuda") * 0.1
    want = rt.attn_paged_i8(kv, r, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for _ in range(20):
        outs.append(rt.attn_paged_i8(kv, r, q, stream=side.cuda_stream))
        torch.full((1 << 18,), float("nan"), device="cuda")        # reuses whatever the current stream freed
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    two = [torch.cuda.Stream() for _ in range(2)]
    ws = [rt.attn_paged_workspace(kv, r, 8) for _ in two]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(20):
        for j in range(2):
            got[j].append(rt.attn_paged_i8(kv, r, q, workspace=ws[j], stream=two[j].cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got[0] + got[1])


def test_prompts_and_single_tokens_on_two_streams_at_once(torch, rt):
    """Two calls on one cache that may overlap, a workspace each: the same bits as one after the other."""
    rows, keys, H, KVH, dh = [300, 1, 200], [300, 2500, 700], 16, 4, 128
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 32)
    mixed, single = rt.KVRows(**plan), rt.KVRows(**ragged(torch, [1, 1, 1], keys, plan["page_table"]), max_rows=1)
    q = torch.randn(sum(rows), H * dh, device="cuda") * dh ** -0.5
    calls = [(mixed, q), (single, q[:3])]
    want = [rt.attn_paged_i8(kv, r, x) for r, x in calls]
    ws = [rt.attn_paged_workspace(kv, r, H) for r, _ in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for j, (r, x) in enumerate(calls):
            got[j].append(rt.attn_paged_i8(kv, r, x, workspace=ws[j], stream=streams[j].cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j]) for j in range(2) for o in got[j])
    kv.check()


def test_refusals_of_the_wrappers(torch, rt):
    kv, plan = pool(torch, rt, [2], [20], 2, 64, 16)
    r = rt.KVRows(**plan)
    q, k = torch.randn(2, 4 * 64, device="cuda"), torch.randn(2, 2 * 64, device="cuda")
    bad = [lambda: rt.attn_paged_i8(kv, r, q[:, :96]), lambda: rt.attn_paged_i8(kv, r, q[:, :192]),
           lambda: rt.attn_paged_i8(kv, r, q[:1]), lambda: rt.attn_paged_i8(kv, r, q.half()),
           lambda: rt.attn_paged_i8(kv, r, q, out=q), lambda: rt.attn_paged_i8(kv, r, q.cpu()),
           lambda: rt.attn_paged_i8(kv, r, q, out=torch.zeros(2, 4 * 64 + 1, device="cuda")[:, 1:]),
           lambda: rt.attn_paged_i8(kv, r, q.t().contiguous().t()),
           lambda: rt.kv_append_i8(kv, r, k, k[:, :64]), lambda: rt.kv_append_i8(kv, r, k[:1], k),
           lambda: rt.kv_append_i8(kv, r, k, k, k_gain=torch.ones(32, device="cuda")),
           lambda: rt.kv_append_i8(kv, r, k, k, table=torch.ones(4, 32, device="cuda")),
           lambda: rt.kv_append_i8(kv, r, k, k, k_gain=torch.ones(64, device="cuda"), eps=-1.0),
           lambda: rt.kv_append_i8(kv, r, k, k, q=q[:, :100]), lambda: rt.kv_append_i8(kv, r, k, k, q=q.double()),
           lambda: rt.kv_read_i8(kv, r, dtype=torch.float16), lambda: rt.kv_read_i8(kv, r, k_out=k[:1]),
           lambda: rt.qk_norm_rope(q, k[:1], 64), lambda: rt.qk_norm_rope(q, k, 48),
           lambda: rt.qk_norm_rope(q, k, 64, table=torch.ones(4, 64, device="cuda")),
           lambda: rt.qk_norm_rope(q, k, 64, pos=torch.zeros(2, device="cuda")),
           lambda: rt.PagedKV(kv.k, kv.v[:, :, :, :32], kv.k_scale, kv.v_scale),
           lambda: rt.PagedKV(kv.k, kv.v, kv.k_scale[:1], kv.v_scale),
           lambda: rt.PagedKV(kv.k.transpose(0, 1), kv.v, kv.k_scale, kv.v_scale),
           lambda: rt.KVRows(plan["row_start"].long(), plan["kv_len"], plan["page_table"], 2),
           lambda: rt.KVRows(plan["row_start"][:1], plan["kv_len"], plan["page_table"], 2),
           lambda: rt.KVRows(plan["row_start"], plan["kv_len"], plan["page_table"], -1)]
    for f in bad:
        with pytest.raises(rt.B2Error):
            f()
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [1, 3, 17])
@pytest.mark.parametrize("KVH,dh", [(3, 16), (2, 64), (2, 128), (1, 256)])
@pytest.mark.parametrize("single", [False, True])
def test_append_norms_without_an_eps(torch, rt, n, KVH, dh, single):
    """eps = 0 is a norm too, for vectors that are not zeros: the block's scale comes from the run's rows alone, however
    many of them a pass holds. `single`: the variant for single rows, by a hint below the truth."""
    g = torch.Generator(device="cuda").manual_seed(n + dh)
    kv = rt.PagedKV.empty(4, 16, KVH, dh)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
    rows = rt.KVRows(**ragged(torch, [n], [n + 2], table), max_rows=int(single))
    k, v = torch.randn(2, n, KVH * dh, device="cuda", generator=g)
    gain = 1 + 0.3 * torch.rand(dh, device="cuda", generator=g)
    rt.kv_append_i8(kv, rows, k, v, k_gain=gain, eps=0.0)
    x = k.reshape(n, KVH, dh).double()
    want = x / x.square().mean(-1, keepdim=True).sqrt() * gain.double()
    got = held(torch, kv, table, 0, n + 2)[0][2:]
    for lo in range(0, n + 2, 16):
        a, b = max(lo - 2, 0), min(lo + 14, n)
        top = want[a:b].abs().amax((0, 2), keepdim=True)
        # half a step of the scale, which is top / 127 up to f32, and what f32 did before the code was chosen
        close(torch, got[a:b], want[a:b], (0.5 * top / 127 * (1 + 1e-5)).expand(b - a, -1, dh) + turn_tol(want[a:b].abs(), dh))
    kv.check()


@pytest.mark.parametrize("H,KVH,dh,rows,keys,cap,hint", [
    (32, 8, 128, [1500, 1, 4, 0, 3], [1500, 6000, 4, 900, 20000], 1 << 17, 0),       # short sequences' rows in an area of their own
    (8, 2, 64, [60, 1, 1, 4], [3000, 6000, 30, 1300], 0, 0),                       # both kinds split, rows numbered in their sequences
    (4, 2, 128, [20, 1, 0, 1, 8], [2000, 6000, 3, 30, 1300], 0, 0),                # both kinds split, by the call's rows
    (48, 2, 64, [3, 1, 40], [5000, 9000, 100], 0, 0), (4, 2, 256, [30, 1, 2], [700, 9000, 5000], 0, 0),
    (16, 4, 128, [1] * 6, [9000, 1, 300, 5000, 513, 2], 0, 1), (8, 2, 80, [33], [9000], 0, 0)])
def test_workspace_is_enough_and_read_only_where_written(torch, rt, H, KVH, dh, rows, keys, cap, hint):
    """Just the bytes asked for, full of NaNs at the start: the outputs are right and nothing behind them is touched."""
    kv, plan = pool(torch, rt, rows, keys, KVH, dh, 64, seed=6)
    if cap:                                                        # a wide table: the capacity, not the keys, is large
        wide = torch.full((len(rows), cap // 64), -1, dtype=torch.int32, device="cuda")
        wide[:, :plan["page_table"].shape[1]] = plan["page_table"]
        plan["page_table"] = wide
    n = sum(rows)
    q = torch.randn(n, H * dh, device="cuda") * dh ** -0.5
    r = rt.KVRows(**plan, max_rows=hint)
    need = rt.attn_paged_workspace(kv, r, H).numel()
    assert need > 0
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
    out = rt.attn_paged_i8(kv, r, q, workspace=ws[:need])
    close(torch, out.reshape(n, H, dh), *attend64(torch, kv, plan, rows, keys, q, H))
    assert bool((ws[need:] == 255).all())
    with pytest.raises(rt.B2Error, match="workspace"):
        rt.attn_paged_i8(kv, r, q, workspace=ws[:need - 16])
    kv.check()


def decode_step_us(torch, rt, n, keys, H, KVH, dh):
    """Device time of an attention call among others with and without max_rows = 1, taken in turn, over caches that do
    not stay in L2 together."""
    g = torch.Generator(device="cuda").manual_seed(n)
    per = -(-keys // 64)
    table = torch.randperm(n * per, device="cuda", generator=g).to(torch.int32).reshape(n, per)
    kvs = [rt.PagedKV.empty(n * per, 64, KVH, dh) for _ in range(3)]
    for kv in kvs:
        for codes, scale in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
            codes.random_(-127, 128, generator=g)
            scale.fill_(0.02)
    q = torch.randn(n, H * dh, device="cuda", generator=g) * dh ** -0.5
    out, best = torch.empty_like(q), [math.inf, math.inf]
    rows = [rt.KVRows(**ragged(torch, [1] * n, [keys] * n, table), max_keys=keys, max_rows=hint) for hint in (1, 0)]
    ws = [rt.attn_paged_workspace(kvs[0], r, H) for r in rows]
    for _ in range(10):
        for j, r in enumerate(rows):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for i in range(12):
                rt.attn_paged_i8(kvs[i % 3], r, q, out=out, workspace=ws[j])
            b.record()
            torch.cuda.synchronize()
            best[j] = min(best[j], a.elapsed_time(b) / 12 * 1e3)
    return best


def test_a_decode_step_without_the_hint(torch, rt):
    """64 single tokens that are not said to be single: a small launch that finds nothing to do, not thousands of CTAs
    (221 against 119 us)."""
    hint, none = decode_step_us(torch, rt, 64, 1152, 32, 32, 128)
    assert none < 1.5 * hint


@pytest.mark.parametrize("heads,dh", [(32, 128), (16, 256)])
def test_single_tokens_behind_the_launch_for_longer_sequences(torch, rt, heads, dh):
    """The kernel of the single tokens is as fast behind the other kernel's (here empty) launch as without it: its loads
    do not suffer from that kernel's use of the SM (152 against 119 us, with d_head 256 169 against 128)."""
    hint, none = decode_step_us(torch, rt, 64, 1152, heads, heads, dh)
    assert none < 1.17 * hint


def test_check_waits_for_calls_on_other_streams(torch, rt):
    """A bad page met by a call that still waits on a side stream is reported, and once."""
    kv, plan = pool(torch, rt, [1], [40], 2, 64, 16)
    plan["page_table"][0, 1] = -1
    r = rt.KVRows(**plan)
    q = torch.randn(1, 2 * 64, device="cuda")
    rt.attn_paged_i8(kv, r, q)                                     # (an earlier report, to be cleared)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(2):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)                         # 0.1 s or so
        rt.attn_paged_i8(kv, r, q, stream=side.cuda_stream)
        with pytest.raises(rt.B2Error, match="page-table entry"):
            kv.check()
        assert side.query()
        kv.check()


@pytest.mark.parametrize("start,bad", [([0, 12, 0, 12], True), ([0, 4, 2, 12], True), ([4, 2, 2, 12], True), ([0, 4, 8, 12], False),
                                       ([3, 3, 3, 3], False), ([-5, 4, 8, 900], False), ([0] * 40 + [6] + [5] * 2, True)])
def test_row_ranges_that_may_overlap_are_reported(torch, rt, start, bad):
    """By append and by read, wherever a start is below the one before it; other odd starts are no error."""
    n = len(start) - 1
    kv = rt.PagedKV.empty(n, 16, 1, 32)
    plan = dict(row_start=torch.tensor(start, dtype=torch.int32, device="cuda"), n_rows=12,
                kv_len=torch.full((n,), 16, dtype=torch.int32, device="cuda"),
                page_table=torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous())
    x = torch.randn(12, 32, device="cuda")
    for hint in (0, 1):
        r = rt.KVRows(**plan, max_rows=hint)
        for call in (lambda: rt.kv_append_i8(kv, r, x, x), lambda: rt.kv_read_i8(kv, r)):
            call()
            if bad:
                with pytest.raises(rt.B2Error, match="overlap"):
                    kv.check()
            kv.check()


def test_outputs_do_not_follow_the_default_dtype(torch, rt):
    """A serving program's default dtype is often bfloat16: caches and outputs that the calls make are f32 all the same."""
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    plan = ragged(torch, [3], [3], table)
    q, k = (torch.randn(3, w, device="cuda") for w in (128, 64))
    torch.set_default_dtype(torch.bfloat16)
    try:
        kv, r = rt.PagedKV.empty(1, 16, 1, 64), rt.KVRows(**plan)
        made = [kv.k_scale, *rt.qk_norm_rope(q, k, 64), rt.kv_append_i8(kv, r, k, k, q=q), rt.attn_paged_i8(kv, r, q), *rt.kv_read_i8(kv, r)]
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(x.dtype is torch.float32 for x in made)
    kv.check()


def test_bounds_beyond_32_bits(torch, rt):
    """A max_keys or max_rows above 2^31 bounds nothing and does not wrap around; such an n_rows is refused."""
    rows, keys = [2], [40]
    kv, plan = pool(torch, rt, rows, keys, 2, 64, 16)
    q = torch.randn(2, 4 * 64, device="cuda") * 0.1
    want, tol = attend64(torch, kv, plan, rows, keys, q, 4)
    for bound in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 16):
        close(torch, rt.attn_paged_i8(kv, rt.KVRows(**plan, max_keys=bound, max_rows=bound), q).reshape(2, 4, 64), want, tol)
        kv.check()
    for n in (2 ** 31, 2 ** 32 + 2):
        with pytest.raises(rt.B2Error):
            rt.KVRows(**{**plan, "n_rows": n})


@pytest.mark.parametrize("factor", [10, 100, 1000])
@pytest.mark.parametrize("n,H,KVH,dh", [(1, 8, 8, 128), (1, 8, 2, 64), (130, 8, 8, 128), (70, 4, 4, 256)])
def test_a_query_channel_that_stands_out(torch, rt, n, H, KVH, dh, factor):
    """One channel `factor` times the others, where the keys have small codes: within the documented rounding, and as the
    documentation says below d_head / 65000 of a half step of the keys there, which moves a score by `half` or less."""
    keys = 1152
    kv, plan = pool(torch, rt, [n], [keys], KVH, dh, 64, seed=3)
    kv.k[..., 5] = 3
    q = torch.randn(n, H, dh, device="cuda") * dh ** -0.5
    q[..., 5] = factor * dh ** -0.5
    out = rt.attn_paged_i8(kv, rt.KVRows(**plan), q.reshape(n, -1)).reshape(n, H, dh)
    want, tol = attend64(torch, kv, plan, [n], [keys], q.reshape(n, -1), H)
    close(torch, out, want, tol)
    # all scores off by at most e move an output by at most (exp(2 e) - 1) times the largest value; the f32 part of the
    # errors is attend64's without its term for held queries
    half = factor * dh ** -0.5 * float(kv.k_scale.nan_to_num(0.0).max()) / 2
    top_v = 127 * float(kv.v_scale.nan_to_num(0.0).max())
    k = held(torch, kv, plan["page_table"], 0, keys)[0].repeat_interleave(H // KVH, 1).transpose(0, 1)
    mag = float((q.double().abs().transpose(0, 1) @ k.abs().transpose(1, 2)).max())
    f32 = (2 * (6 * math.sqrt(dh) + 8) * mag + 2 * 104 + 16 + 18 * math.sqrt(keys)) * U
    assert float((out.double() - want).abs().max()) <= top_v * (math.expm1(2 * half * dh / 65000) + f32)
    kv.check()


def test_the_default_stream_by_its_handle(torch, rt):
    """stream=0 is the default stream, also where another one is current: calls stand behind what was queued there."""
    kv, plan = pool(torch, rt, [1, 1], [300, 40], 2, 64, 16)
    r = rt.KVRows(**plan)
    new = torch.randn(2, 4 * 64, device="cuda") * 0.1
    want, tol = attend64(torch, kv, plan, [1, 1], [300, 40], new, 4)
    q, out, ws = torch.zeros_like(new), torch.zeros_like(new), rt.attn_paged_workspace(kv, r, 4)   # (an allocation would wait)
    default, side = torch.cuda.default_stream(), torch.cuda.Stream()
    assert default.cuda_stream == 0
    rt.attn_paged_i8(kv, r, q, out=out, workspace=ws)              # (loading a kernel would wait, too)
    torch.cuda.synchronize()
    with torch.cuda.stream(default):
        torch.cuda._sleep(200_000_000)
        q.copy_(new)
    with torch.cuda.stream(side):
        rt.attn_paged_i8(kv, r, q, out=out, workspace=ws, stream=0)
    torch.cuda.synchronize()
    close(torch, out.reshape(2, 4, 64), want, tol)


def test_a_captured_step_behind_other_streams(torch, rt):
    """Captured with a fork and a join: one stream fills the keys and values, another the queries; the calls stand behind
    both, and a copy of the outputs behind them, in every replay."""
    H, KVH, dh = 8, 2, 128
    table = torch.arange(20, dtype=torch.int32, device="cuda").reshape(2, 10)
    kv = rt.PagedKV.empty(20, 16, KVH, dh)
    plan = ragged(torch, [1, 30], [1, 30], table)
    r = rt.KVRows(**plan)
    src = [torch.randn(31, w * dh, device="cuda") for w in (H, KVH, KVH)]
    q, k, v = (torch.zeros_like(x) for x in src)
    out, copy = torch.zeros(31, H * dh, device="cuda"), torch.zeros(31, H * dh, device="cuda")
    ws = rt.attn_paged_workspace(kv, r, H)
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q.zero_()
            q.copy_(src[0])
        k.copy_(src[1])
        v.copy_(src[2])
        main.wait_stream(side)
        rt.kv_append_i8(kv, r, k, v)
        rt.attn_paged_i8(kv, r, q, out=out, workspace=ws)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            copy.copy_(out)
        main.wait_stream(side)

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        for x in src:
            x.copy_(torch.randn_like(x) * 0.2)
        copy.zero_()
        graph.replay()
        close(torch, copy.reshape(31, H, dh), *attend64(torch, kv, plan, [1, 30], [1, 30], src[0], H))
    kv.check()


def test_in_place_and_side_by_side_in_one_buffer(torch, rt):
    """Queries rewritten where they lie, outputs in columns of the buffer that holds the inputs: as with outputs of their own."""
    H, KVH, dh = 4, 2, 64
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    tab = table64(torch, 64, dh)
    r = rt.KVRows(**ragged(torch, [40], [40], table))
    buf = torch.randn(40, (2 * H + 2 * KVH) * dh, device="cuda")
    q, k, v, out = (x for x in buf.split([H * dh, KVH * dh, KVH * dh, H * dh], 1))
    kv, other = rt.PagedKV.empty(4, 16, KVH, dh), rt.PagedKV.empty(4, 16, KVH, dh)
    qo = rt.kv_append_i8(other, r, k, v, table=tab, q=q, q_scale=dh ** -0.5)
    want = rt.attn_paged_i8(other, r, qo)
    rt.kv_append_i8(kv, r, k, v, table=tab, q=q, q_scale=dh ** -0.5, q_out=q)
    rt.attn_paged_i8(kv, r, q, out=out)
    assert torch.equal(q, qo) and torch.equal(out, want) and torch.equal(kv.k, other.k) and torch.equal(kv.v, other.v)
