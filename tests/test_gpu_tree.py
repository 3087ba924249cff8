"""Trees of drafted tokens: attn_tree_i8, tree_accept and kv_append_kept_i8 against plain implementations in 64 bits, and a
whole verification step.

Tolerances. u = 2^-24 is half a step of f32. A score is off by at most 4 u of its terms' magnitude for the roundings of each
factor, 2 u for each of the d / 8 steps of 16 elements that a matrix unit adds (it cuts off, which is at most two half
steps), and a few more: (d / 4 + 24) u. A probability is off by twice the worst of that in its row, its exponent's argument
(two u for each unit of the row's spread) and a few u; the sum over the keys 6 sqrt(n) u, twice (numerator and
denominator); weights 4 u, 32 u for a tile's sums, one for each addition of a tile (n / 128): together
2 e + (2 spread + 80 + 12 sqrt(n) + n / 128) u of sum p |v|. Weights below 2^-40 of the largest may be dropped: that much of
the largest value scale on top."""
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


# ------------------------------------------------------------------ inputs and plain implementations
def parents_of(rng, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    return [-1] + [rng.randrange(j) for j in range(1, n)] if n else []


def make(torch, rt, rows, cached, H, KVH, dh, page, seed=0, pad=0, kind="tree", wide=0, **hints):
    """A cache of `cached` keys a sequence in scattered pages (scales that no key uses are NaN, table entries past the keys
    nonsense) and drafted rows with trees. Returns a dict."""
    import random
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-k // page) for k in cached]
    n_pages, most = sum(need) + 2, max(need + [0]) + 5
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(cached), most), -12345, dtype=torch.int32, device="cuda")
    kv = rt.PagedKV.empty(n_pages, page, KVH, dh)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    for name in ("k", "v"):
        getattr(kv, name).copy_(torch.randint(-127, 128, kv.k.shape, device="cuda", generator=g, dtype=torch.int8))
        scale = torch.full_like(kv.k_scale, float("nan"))
        for s, k in enumerate(cached):
            for b in range(-(-k // 16)):
                scale[int(table[s, b * 16 // page]), :, b * 16 % page // 16] = 0.005 + 0.02 * torch.rand(KVH, device="cuda", generator=g)
        getattr(kv, name + "_scale").copy_(scale)
    n = sum(rows) + pad
    parents = [parents_of(rng, r, kind) for r in rows]
    seen = sum((rt.tree_seen(p) for p in parents), []) + [-1] * pad
    start = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    qkv = torch.randn(n, (H + 2 * KVH) * dh + wide, device="cuda", generator=g)
    q = qkv[:, :H * dh]
    q *= dh ** -0.5
    c = dict(kv=kv, table=table, rows=rows, cached=list(cached), H=H, KVH=KVH, dh=dh, parents=parents, pad=pad, q=q,
             k=qkv[:, H * dh:(H + KVH) * dh], v=qkv[:, (H + KVH) * dh:(H + 2 * KVH) * dh])
    c["tree"] = rt.TreeRows(start, torch.tensor(cached, dtype=torch.int32, device="cuda"), table,
                            torch.tensor(seen, dtype=torch.int64, device="cuda"), n_rows=n, **hints)
    return c


def held(torch, kv, table, s, n):
    """(k, v, there) of the first n cached keys of sequence s in 64 bits, [n, kv_heads, d]; keys on bad pages are not there."""
    j = torch.arange(n, device="cuda")
    page = table[s].long()[j // kv.page_size] if n else j
    there = (page >= 0) & (page < kv.n_pages)
    page = torch.where(there, page, 0)
    off = j % kv.page_size
    out = [x[page, :, off].double() * sc[page, :, off // 16].double()[..., None] for x, sc in ((kv.k, kv.k_scale), (kv.v, kv.v_scale))]
    return (*out, there)


def attend64(torch, c, capacity=None):
    """(out, tolerance) [n_rows, H, d] in 64 bits, of the rows that belong to a sequence."""
    kv, H, KVH, d, tree = c["kv"], c["H"], c["KVH"], c["dh"], c["tree"]
    G, outs, tols, a = H // KVH, [], [], 0
    for s, (r, n) in enumerate(zip(c["rows"], c["cached"])):
        if r == 0:
            continue
        n = min(n, capacity or n)
        ck, cv, there = held(torch, kv, c["table"], s, n)
        new = slice(a, a + r)
        k = torch.cat((ck, c["k"][new].reshape(r, KVH, d).double())).repeat_interleave(G, 1).transpose(0, 1)   # [H, n + r, d]
        v = torch.cat((cv, c["v"][new].reshape(r, KVH, d).double())).repeat_interleave(G, 1).transpose(0, 1)
        bits = (tree.seen[new, None] >> torch.arange(r, device="cuda") & 1).bool()
        sees = torch.cat((there[None].expand(r, -1), bits), 1)[None]                                          # [1, r, n + r]
        q = c["q"][new].reshape(r, H, d).double().transpose(0, 1)
        score = (q @ k.transpose(1, 2)).masked_fill(~sees, -math.inf)
        none = ~sees.any(-1, keepdim=True)
        p = torch.where(none, 0.0, torch.softmax(score.masked_fill(none, 0.0), -1))
        p = torch.where(sees, p, 0.0)
        vz = torch.where(sees.any(1)[0, :, None], v, 0.0)              # what nobody sees, whatever it holds
        out = p @ vz
        mag = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(~sees, 0.0)
        e = (d / 4 + 24) * U * mag.amax(-1, keepdim=True)
        spread = (score.amax(-1, keepdim=True) - score.masked_fill(~sees, math.inf).amin(-1, keepdim=True)).nan_to_num(0.0, 0.0, 0.0).clamp(0, 100)
        m = n + r
        tol = (2 * e + (2 * spread + 80 + 12 * math.sqrt(m) + m / 128) * U) * (p @ vz.abs())
        tol = tol + 2.0 ** -40 * m * vz.abs().amax() if m else tol
        outs.append(out.transpose(0, 1))
        tols.append(tol.transpose(0, 1))
        a += r
    return torch.cat(outs), torch.cat(tols)


def close(got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)                             # a NaN is bad
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max()))


def attend(rt, c, **kw):
    return rt.attn_tree_i8(c["kv"], c["tree"], c["q"], c["k"], c["v"], **kw)


def check_attention(torch, rt, c, capacity=None):
    T, H, d = sum(c["rows"]), c["H"], c["dh"]
    out = torch.full((T + c["pad"], H * d), 7.0, device="cuda")
    attend(rt, c, out=out)
    want, tol = attend64(torch, c, capacity)
    close(out[:T].reshape(T, H, d), want, tol)
    assert bool((out[T:] == 7.0).all())                            # rows behind the last sequence
    return out


# ------------------------------------------------------------------ attention
SHAPES = [  # rows, cached, H, KVH, dh, page
    ([1], [0], 1, 1, 16, 16),
    ([1], [1], 2, 1, 64, 16),
    ([3], [15], 4, 4, 128, 16),
    ([5], [639], 32, 32, 128, 16),
    ([64], [128], 8, 1, 64, 32),
    ([64], [1000], 4, 2, 128, 64),
    ([64, 1, 33], [300, 0, 17], 6, 2, 128, 16),
    ([0, 7, 0, 16, 2], [5, 129, 0, 4097, 256], 16, 4, 128, 128),
    ([13], [2000], 8, 2, 80, 16),
    ([9, 60], [127, 383], 14, 7, 96, 32),
    ([17], [515], 4, 1, 256, 16),
    ([40, 3], [100, 900], 6, 2, 208, 64),
    ([8] * 20, list(range(100, 2100, 100)), 4, 4, 64, 16),
    ([11], [20000], 4, 2, 64, 128),
    ([30], [9000], 16, 1, 128, 1024),
    ([64] * 3, [700, 1, 64], 32, 2, 48, 16),
    ([2] * 300, [20] * 300, 2, 1, 32, 16),
]


@pytest.mark.parametrize("rows,cached,H,KVH,dh,page", SHAPES)
def test_attention(torch, rt, rows, cached, H, KVH, dh, page):
    c = make(torch, rt, rows, cached, H, KVH, dh, page, seed=sum(rows) + dh)
    check_attention(torch, rt, c)
    c["kv"].check()


@pytest.mark.parametrize("kind", ["chain", "star", "tree"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64])
def test_kinds_of_trees(torch, rt, kind, n):
    check_attention(torch, rt, make(torch, rt, [n, 5], [40, 0], 4, 2, 64, 16, seed=n, kind=kind, max_keys=64))


@pytest.mark.parametrize("hints", [dict(), dict(max_rows=64), dict(max_rows=12), dict(max_keys=700), dict(max_rows=12, max_keys=611)])
def test_hints_do_not_change_what_comes_out(torch, rt, hints):
    c = make(torch, rt, [12, 0, 7, 1], [611, 20, 64, 300], 8, 2, 128, 16, seed=5, pad=3, wide=8, **hints)
    check_attention(torch, rt, c)


@pytest.mark.parametrize("dh", [64, 128, 256])
def test_any_mask(torch, rt, dh):
    """Words that are no tree: later rows, not itself, bits past the rows, nothing."""
    c = make(torch, rt, [30, 64, 3], [50, 0, 0], 4, 2, dh, 16, seed=dh)
    g = torch.Generator(device="cuda").manual_seed(1)
    c["tree"].seen.copy_(torch.randint(-(1 << 62), 1 << 62, (97,), device="cuda", generator=g) * 2)
    c["tree"].seen[3] = 0
    c["tree"].seen[40] = 0                                         # sees nothing at all: zeros
    c["tree"].seen[41] = -(1 << 63)
    c["tree"].seen[95] = 1 << 5                                    # a bit past the rows: nothing either
    out = check_attention(torch, rt, c)
    assert not out[40].any() and not out[95].any() and out[41].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_what_is_not_finite_stays_with_who_sees_it(torch, rt, which, bad):
    """Row 4 (and its descendants) see a NaN; the others do not, though it lies in their tile."""
    c = make(torch, rt, [20, 20], [100, 30], 4, 2, 128, 16, seed=3)
    c[which][4, 70] = bad                                          # KV head 0 (d 70), query head 0
    out = attend(rt, c).reshape(40, 4, 128)
    sees = [(rt.tree_seen(c["parents"][0])[i] >> 4) & 1 == 1 for i in range(20)]
    assert 1 < sum(sees) < 20
    want, tol = attend64(torch, {**c, which: c[which].nan_to_num(0.0, 0.0, 0.0)})
    for i in range(40):
        for h in range(4):
            hit = (i == 4 and h == 0) if which == "q" else (i < 20 and sees[i] and h < 2)
            if hit:
                assert bool(out[i, h].isnan().all()), (i, h)
            else:
                close(out[i, h], want[i, h], tol[i, h])


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_poisoned_block_is_seen_by_its_sequence_and_head(torch, rt, which):
    c = make(torch, rt, [6, 6], [300, 300], 4, 2, 128, 16, seed=4)
    getattr(c["kv"], which)[int(c["table"][0, 7]), 1, 0] = float("nan")
    out = attend(rt, c).reshape(12, 4, 128)
    assert bool(out[:6, 2:].isnan().all()) and not bool(out[:6, :2].isnan().any()) and not bool(out[6:].isnan().any())


def test_rows_of_very_different_sizes(torch, rt):
    """Queries 1e-20 and 1e20 times the others (their softmax is flat or one key's), large and tiny drafted keys and values."""
    c = make(torch, rt, [16], [200], 4, 2, 128, 16, seed=6)
    c["q"][3] *= 1e-20
    c["k"][5] *= 1e-6
    c["v"][6] *= 1e-6
    c["v"][7] *= 3e3
    c["v"][:, 64] *= 1e-4
    check_attention(torch, rt, c)
    want = attend(rt, c)[:3].clone()
    c["q"][9] *= 1e20                                              # finite: others do not notice
    assert torch.equal(attend(rt, c)[:3], want)


def test_small_and_large_value_scales(torch, rt):
    for f in (1e-12, 1e12, 1e-30):
        c = make(torch, rt, [10], [400], 4, 2, 64, 16, seed=7)
        c["kv"].v_scale *= f
        c["v"].mul_(f)
        check_attention(torch, rt, c)


def attend64_by_sum(torch, c, rows, bits):
    """(out, tolerance) [len(rows), H, d] in 64 bits of rows of one sequence (c has no other), where value scales differ by up
    to 2^bits. The tolerance is attend64's without the dropped weights, which are relative to all values there are; instead
    a weight may be off by 2^-30 of the largest power of two in p |v| over what the row sees (half a step of the smaller f16,
    2^-25, where the largest is brought to 2^5 or more), that is 2^-29 of its largest p |v| for each of its keys; and the exponents' arguments lie up to `bits`
    from their base, which is rounded to u of itself, numerator and denominator."""
    kv, H, KVH, d, tree = c["kv"], c["H"], c["KVH"], c["dh"], c["tree"]
    (r,), (n,), G = c["rows"], c["cached"], H // KVH
    ck, cv, there = held(torch, kv, c["table"], 0, n)
    k = torch.cat((ck, c["k"][:r].reshape(r, KVH, d).double())).repeat_interleave(G, 1).transpose(0, 1)      # [H, n + r, d]
    v = torch.cat((cv, c["v"][:r].reshape(r, KVH, d).double())).repeat_interleave(G, 1).transpose(0, 1)
    mine = torch.tensor(rows, device="cuda")
    words = tree.seen[mine, None] >> torch.arange(r, device="cuda") & 1
    sees = torch.cat((there[None].expand(len(rows), -1), words.bool()), 1)[None]
    q = c["q"][:r].reshape(r, H, d).double()[mine].transpose(0, 1)
    score = (q @ k.transpose(1, 2)).masked_fill(~sees, -math.inf)
    p = torch.softmax(score, -1)
    mag = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(~sees, 0.0)
    e = (d / 4 + 24) * U * mag.amax(-1, keepdim=True)
    top = score.amax(-1, keepdim=True)
    spread = (top - score.masked_fill(~sees, math.inf).amin(-1, keepdim=True)).clamp(0, 100)
    m = n + r
    tol = (2 * e + (2 * spread + 2 * bits + 80 + 12 * math.sqrt(m) + m / 128) * U) * (p @ v.abs())
    tol = tol + m * 2.0 ** -29 * (p * v.abs().amax(-1)[:, None]).amax(-1, keepdim=True)
    return (p @ v).transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("cached", [0, 30, 700])
@pytest.mark.parametrize("factor", [1e4, 1e6, 1e10, 1e20])
@pytest.mark.parametrize("H,KVH,dh", [(4, 2, 128), (4, 4, 64), (2, 1, 256), (16, 2, 64)])
def test_large_values_of_a_row_cost_only_who_sees_it(torch, rt, H, KVH, dh, cached, factor):
    """A star whose row 3 has values far above the others': its siblings do not see it."""
    c = make(torch, rt, [9], [cached], H, KVH, dh, 16, seed=cached + dh, kind="star")
    c["v"][3] *= factor
    out = attend(rt, c).reshape(9, H, dh)
    others = [i for i in range(9) if i != 3]
    want, tol = attend64_by_sum(torch, c, others, math.log2(factor) + 4)
    close(out[others], want, tol)
    want, tol = attend64_by_sum(torch, c, [3], math.log2(factor) + 4)
    close(out[3:4], want, tol)


@pytest.mark.parametrize("where", [0, 17, 40])
@pytest.mark.parametrize("bits", [14, 20, 40, 70])
@pytest.mark.parametrize("away", [0.0, 0.35, 2.0])
@pytest.mark.parametrize("H,KVH,dh", [(4, 2, 128), (16, 2, 64)])
def test_large_values_of_cached_keys(torch, rt, H, KVH, dh, away, bits, where):
    """A block of the cache with value scales 2^bits times the others': at a probability of nothing, at one that about makes up
    for it, and at the others' own."""
    c = make(torch, rt, [8], [700], H, KVH, dh, 16, seed=bits + where)
    kv = c["kv"]
    c["q"].copy_(dh ** -0.5 * (1 + 0.1 * c["q"] * dh ** 0.5))
    page = int(c["table"][0, where])
    kv.v_scale[page, :, 0] *= 2.0 ** bits
    if away:                                                       # scores of about -away * bits * 2 nats
        kv.k[page] = -127
        kv.k_scale[page, :, 0] = away * bits * 2 / (127 * dh ** 0.5)
    want, tol = attend64_by_sum(torch, c, list(range(8)), bits + 4)
    close(attend(rt, c).reshape(8, H, dh), want, tol)


@pytest.mark.parametrize("small,large", [(2.0 ** -60, 1.0), (2.0 ** -30, 2.0 ** 40), (0.0, 1.0)])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("cached", [300, 5000])
def test_values_that_grow_or_shrink_along_a_sequence(torch, rt, cached, first, small, large):
    """Half of the cached keys have tiny values (or none): their probability counts all the same, in one split and in several."""
    c = make(torch, rt, [8], [cached], 8, 2, 64, 16, seed=cached)
    half = c["table"][0, :-(-cached // 16)].long()
    half = half[:len(half) // 2] if first else half[len(half) // 2:]
    c["kv"].v_scale *= large
    c["kv"].v_scale[half] *= small / large
    c["v"].mul_(large)
    want, tol = attend64_by_sum(torch, c, list(range(8)), 74)
    close(attend(rt, c).reshape(8, 8, 64), want, tol)


@pytest.mark.parametrize("cached", [200, 5000])
@pytest.mark.parametrize("code", [64, 100])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 27, 2.0 ** 32, 2.0 ** 66])
def test_equal_scores_of_any_size(torch, rt, cached, code, size):
    """All keys the same, scores of about +size or -size: the mean of the values, whatever the parts that they are summed in.
    With codes of +-64 the sum of products is a power of two, so a score in base 2 is log2 e (as f32 has it) times one: exact
    in f32, and every weight is the same. With others a score is rounded in an item's first tile (which finds the base) and
    not in the next, where it is multiplied and subtracted in one: arguments differ by up to u of the score in base 2, a
    weight by that times ln 2, numerator and denominator: 2 u size more of sum p |v|, which from 2^24 on says only that what
    comes out is finite and no larger than the values."""
    c = make(torch, rt, [6], [cached], 4, 2, 64, 16, seed=cached)
    kv = c["kv"]
    kv.k.copy_(torch.where(torch.arange(64, device="cuda") % 2 == 0, code, -code))
    kv.k_scale.fill_(2.0 ** -7)
    c["q"].copy_(torch.where(torch.arange(256, device="cuda") % 2 == 0, 1.0, -1.0) * (size / 32))
    c["q"][3:] *= -1
    c["tree"].seen.zero_()                                         # the cached keys alone
    _, v, _ = held(torch, kv, c["table"], 0, cached)
    v = v.repeat_interleave(2, 1)
    want, mag = v.mean(0), v.abs().mean(0)
    tol = (80 + 12 * math.sqrt(cached) + cached / 128) * U * mag + 2.0 ** -29 * v.abs().amax()
    if code != 64:
        tol = tol + min(4 * U * size, 2.0) * v.abs().amax(0)       # (a size of 2 codes / 64: 2 u size and a half)
    close(attend(rt, c).reshape(6, 4, 64), want.expand(6, -1, -1), tol.expand(6, -1, -1))


@pytest.mark.parametrize("cached", [200, 5000])
@pytest.mark.parametrize("bits", [0, 6, 35])
@pytest.mark.parametrize("size", [1e8, 1e9, 1e12, 1e20])
def test_huge_scores(torch, rt, cached, bits, size):
    """One key has it all: its values come out. Beside scores above 2^24 their base cannot follow the exponents of value scales
    exactly (2^-bits to 2^bits here): it is off by no more than their range, 2 bits + 1, and so many bits the weights lose of the
    30 that they have below the largest. With more than those it is tested that nothing overflows."""
    c = make(torch, rt, [6], [cached], 4, 2, 64, 16, seed=cached)
    kv = c["kv"]
    kv.v_scale *= 2.0 ** torch.randint(-bits, bits + 1, kv.v_scale.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    c["q"] *= size
    out = attend(rt, c).reshape(6, 4, 64)
    want, _ = attend64_by_sum(torch, c, list(range(6)), 74)
    if bits < 12:
        close(out, want, 32 * U * want.abs() + 2.0 ** (2 * bits + 1 - 29) * want.abs().amax(-1, keepdim=True))
    else:
        _, v, _ = held(torch, kv, c["table"], 0, cached)
        assert bool((out.abs() <= 1.01 * max(float(v.abs().amax()), float(c["v"].abs().amax()))).all())


def test_pages_outside_the_pool_are_left_out(torch, rt):
    c = make(torch, rt, [10, 12], [400, 500], 8, 2, 128, 16, seed=8)
    c["table"][0, 3], c["table"][0, 24], c["table"][1, 0], c["table"][1, 8] = -1, 1 << 30, c["kv"].n_pages, -(1 << 31)
    check_attention(torch, rt, c)
    with pytest.raises(rt.B2Error, match="page-table"):
        c["kv"].check()
    c["kv"].check()
    c["table"][:] = -1                                             # the drafted rows alone are left
    check_attention(torch, rt, c)


def test_keys_past_the_capacity_are_left_out(torch, rt):
    c = make(torch, rt, [10], [400], 4, 2, 64, 16, seed=9, max_keys=333)
    check_attention(torch, rt, c, capacity=333)
    with pytest.raises(rt.B2Error, match="capacity"):
        c["kv"].check()


def test_more_rows_than_a_tree_can_have(torch, rt):
    c = make(torch, rt, [10, 64, 10], [100, 50, 30], 4, 2, 64, 16, seed=10)
    c["tree"].row_start.copy_(torch.tensor([0, 10, 75, 84], dtype=torch.int32))      # 65 rows
    out = torch.full((84, 256), 7.0, device="cuda")
    attend(rt, c, out=out)
    with pytest.raises(rt.B2Error, match="more drafted rows"):
        c["kv"].check()
    assert bool((out[10:75] == 7.0).all())
    want, tol = attend64(torch, c)
    close(out[:10].reshape(10, 4, 64), want[:10], tol[:10])


def test_row_ranges_that_make_no_sense(torch, rt):
    """Starts below zero, falling or past the rows: no fault, and a sound sequence beside them is right."""
    c = make(torch, rt, [10, 5, 5, 5], [100, 50, 30, 20], 4, 2, 64, 16, seed=11)
    want, tol = attend64(torch, c)
    for starts in ([0, 10, 3, -7, 100], [0, 10, 1 << 30, 5, 2], [0, 10, 10, 10, 1 << 31 - 1]):
        c["tree"].row_start.copy_(torch.tensor([x & 0x7fffffff if x > 0 else x for x in starts], dtype=torch.int32))
        out = attend(rt, c)
        torch.cuda.synchronize()
        if starts[1:4] == [10, 10, 10]:
            close(out[:10].reshape(10, 4, 64), want[:10], tol[:10])
        c["kv"].err.zero_()
    c["tree"].kv_len.copy_(torch.tensor([-5, 1 << 30, 30, 20], dtype=torch.int32))
    attend(rt, c)
    torch.cuda.synchronize()


def test_strided_rows_and_two_streams(torch, rt):
    """Slices of a fused projection, written into a slice; a call on another stream at the same time, its own workspace."""
    a = make(torch, rt, [20, 3], [700, 900], 8, 2, 128, 16, seed=12, wide=12)
    b = make(torch, rt, [5] * 6, [300] * 6, 8, 8, 64, 32, seed=13)
    big = torch.full((25, 3 * 8 * 128), 7.0, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        attend(rt, a, out=big[1:24, 1024:2048])
        outs.append(attend(rt, b, stream=s.cuda_stream))
    torch.cuda.synchronize()
    want, tol = attend64(torch, a)
    close(big[1:24, 1024:2048].reshape(23, 8, 128), want, tol)
    want, tol = attend64(torch, b)
    for o in outs:
        close(o.reshape(30, 8, 64), want, tol)
    big[1:24, 1024:2048] = 7.0
    assert bool((big == 7.0).all())


def test_captured_calls_replay_with_new_lengths_and_trees(torch, rt):
    """Two graphs with a workspace each, replayed in turn; the second time with other lengths, pages and words."""
    cs = [make(torch, rt, [12, 5, 0, 9], [500, 1100, 7, 64], 8, 2, 128, 16, seed=14 + i, pad=2, max_rows=32) for i in range(2)]
    gs = []
    for c in cs:
        c["out"] = torch.full((28, 1024), 7.0, device="cuda")
        ws = rt.attn_tree_workspace(c["kv"], c["tree"], 8)
        attend(rt, c, out=c["out"], workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attend(rt, c, out=c["out"], workspace=ws)
        gs.append((g, ws))
    for rnd in range(2):
        if rnd:
            for c in cs:
                c["rows"], c["cached"] = [3, 0, 20, 3], [480, 1000, 3, 60]
                seen = sum((rt.tree_seen(parents_of(__import__("random").Random(9), r, "tree")) for r in c["rows"]), []) + [-1] * 2
                c["tree"].seen.copy_(torch.tensor(seen, dtype=torch.int64))
                c["tree"].kv_len.copy_(torch.tensor(c["cached"], dtype=torch.int32))
                c["tree"].row_start.copy_(torch.tensor([0] + c["rows"]).cumsum(0).to(torch.int32))
        for g, _ in gs:
            g.replay()
        torch.cuda.synchronize()
        for c in cs:
            want, tol = attend64(torch, c)
            close(c["out"][:26].reshape(26, 8, 128), want, tol)
            assert bool((c["out"][26:] == 7.0).all())


def test_same_bits_every_time(torch, rt):
    for KVH, dh in ((8, 128), (1, 64)):
        c = make(torch, rt, [16, 40], [3000, 777], 8, KVH, dh, 16, seed=15)
        out = attend(rt, c)
        for _ in range(5):
            assert torch.equal(out, attend(rt, c))


def test_what_behind_a_call_reads_and_writes_is_in_order(torch, rt):
    """The launch before writes the drafted rows, the one behind overwrites them."""
    c = make(torch, rt, [16] * 8, [600] * 8, 8, 2, 128, 16, seed=16)
    want, tol = attend64(torch, c)
    keep = {n: c[n].clone() for n in "qkv"}
    for _ in range(10):
        for n in "qkv":
            c[n].zero_()
            c[n].copy_(keep[n])
        out = attend(rt, c)
        for n in "qkv":
            c[n].fill_(float("nan"))
        close(out.reshape(128, 8, 128), want, tol)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dh,KVH", [(64, 1), (128, 4), (256, 2)])
def test_what_is_not_finite_in_calls_with_splits(torch, rt, dh, KVH, bad):
    """A query and a drafted value: the partial results of everybody else join to what they were."""
    c = make(torch, rt, [12], [6000], 4, KVH, dh, 16, seed=dh)
    assert rt.attn_tree_workspace(c["kv"], c["tree"], 4).numel() > 0
    want, tol = attend64(torch, c)
    c["q"][5, dh + 3] = bad                                        # head 1
    c["v"][2, 7] = bad                                             # KV head 0
    out = attend(rt, c).reshape(12, 4, dh)
    words = rt.tree_seen(c["parents"][0])
    for i in range(12):
        for h in range(4):
            if (i == 5 and h == 1) or (words[i] >> 2 & 1 and h < 4 // KVH):
                assert bool(out[i, h].isnan().all()), (i, h)
            else:
                close(out[i, h], want[i, h], tol[i, h])


def test_threads_with_attention_and_acceptance(torch, rt):
    """Threads on streams of their own, each with all the shapes of the kernel, none with a workspace made before."""
    import threading
    cases = [make(torch, rt, rows, cached, H, KVH, dh, 16, seed=i) for i, (rows, cached, H, KVH, dh) in enumerate(
        (([5], [3000], 4, 4, 64), ([40, 3], [900, 20], 4, 1, 64), ([9], [500], 4, 4, 128), ([33], [2500], 8, 2, 128), ([4], [700], 2, 2, 256),
         ([30], [900], 2, 1, 208)))]
    want = [attend64(torch, c) for c in cases]
    accepts = [accept_case(torch, rt, [9, 3], 5000, seed=i) for i in range(len(cases))]
    tokens = [torch.tensor(a[4], dtype=torch.int32, device="cuda") for a in accepts]
    kept = [rt.tree_accept(a[0], a[1], t).rows.tolist() for a, t in zip(accepts, tokens)]
    torch.cuda.synchronize()
    got, failed = [[] for _ in cases], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for n in range(18):
                    j = (i + n) % len(cases)
                    k = rt.tree_accept(accepts[i][0], accepts[i][1], tokens[i])
                    got[i].append((j, attend(rt, cases[j]), k))
            s.synchronize()
        except Exception as e:                                     # noqa: BLE001 (told by the assertion)
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i, outs in enumerate(got):
        assert len(outs) == 18
        for j, out, k in outs:
            c = cases[j]
            close(out.reshape(sum(c["rows"]), c["H"], c["dh"]), *want[j])
            assert k.rows.tolist() == kept[i]


# ------------------------------------------------------------------ acceptance
def accept_plain(parents, tokens, ids):
    path, at = [], 0 if parents else -1
    while at >= 0:
        path.append(at)
        at = next((j for j in range(len(parents)) if parents[j] == at and tokens[j] == ids[path[-1]]), -1)
    return path


def first_max(row):
    best = 0
    for i, x in enumerate(row):
        if x > row[best]:
            best = i
    return best


def accept_case(torch, rt, rows, vocab, seed=0, pad=0, luck=0.8, wide=0):
    import random
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(rows) + pad
    logits = (torch.randn(n, vocab + wide, device="cuda", generator=g) * 3).bfloat16().float()[:, :vocab]
    parents = [parents_of(rng, r, "tree") for r in rows]
    seen = sum((rt.tree_seen(p) for p in parents), []) + [-1] * pad
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    tree = rt.TreeRows(torch.tensor(start, dtype=torch.int32, device="cuda"),
                       torch.tensor([10 * (s + 1) for s in range(len(rows))], dtype=torch.int32, device="cuda"),
                       torch.zeros(len(rows), 1, dtype=torch.int32, device="cuda"),
                       torch.tensor(seen, dtype=torch.int64, device="cuda"), n_rows=n)
    ids = logits.argmax(-1).tolist()                               # (ties: the tests that have them look themselves)
    tokens = [rng.randrange(vocab) for _ in range(n)]
    for a, p in zip(start, parents):
        for j, up in enumerate(p):
            if up >= 0 and rng.random() < luck:
                tokens[a + j] = ids[a + up]
    return tree, logits, parents, start, tokens


def check_acceptance(torch, rt, tree, logits, parents, start, tokens, kept=None):
    ids = [first_max(r) for r in logits.tolist()] if logits.numel() < 200000 else None
    if ids is None:                                                # the first of the largest ones
        top = logits.amax(-1, keepdim=True)
        ids = torch.where(logits == top, torch.arange(logits.shape[1], device="cuda"), logits.shape[1]).amin(-1).tolist()
    cached = tree.kv_len.tolist()
    tok = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    k = rt.TreeKept(tree) if kept is None else kept
    k.rows.fill_(-7)
    k.ids.fill_(-7)
    assert rt.tree_accept(tree, logits, tok, k) is k
    paths = [accept_plain(p, tokens[a:], ids[a:]) for p, a in zip(parents, start)]
    flat = [a + i for p, a in zip(paths, start) for i in p]
    rest = [-7] * (tree.n_rows - len(flat))
    sums = [0]
    for p in paths:
        sums.append(sums[-1] + len(p))
    assert k.start.tolist() == sums
    assert k.kv_len.tolist() == [c + len(p) for c, p in zip(cached, paths)]
    assert k.rows.tolist() == flat + rest and k.ids.tolist() == [ids[r] for r in flat] + rest
    tree.check()
    return paths


@pytest.mark.parametrize("vocab", [1, 2, 31, 256, 1000, 4099, 50257])
@pytest.mark.parametrize("rows", [[1], [8], [64], [0, 5, 0, 33, 64, 1]])
def test_accepted_paths(torch, rt, rows, vocab):
    paths = check_acceptance(torch, rt, *accept_case(torch, rt, rows, vocab, seed=vocab + len(rows), pad=2))
    assert vocab < 256 or rows == [1] or max(map(len, paths)) > 1


def test_many_sequences(torch, rt):
    rows = [(i * 7) % 20 for i in range(1500)]
    check_acceptance(torch, rt, *accept_case(torch, rt, rows, 12, seed=1, pad=5))


def test_more_rows_than_a_grid_dimension_has(torch, rt):
    """66000 rows: more than the 65535 that the second dimension of a grid can count."""
    check_acceptance(torch, rt, *accept_case(torch, rt, [60] * 1100, 3, seed=3, pad=1))


def test_strided_logits(torch, rt):
    check_acceptance(torch, rt, *accept_case(torch, rt, [9, 3], 1001, seed=2, wide=2))


def test_ties_infinities_and_nan(torch, rt):
    """The first of equal logits; -0 is 0; a NaN never wins, except that one in front of a row leaves 0."""
    inf, nan = float("inf"), float("nan")
    cases = [[1, 5, 5, 2], [-0.0, 0.0, -1, 0], [-inf] * 4, [nan] * 4, [-inf, nan, -inf, nan], [nan, 3, 4, 1], [1, nan, 7, nan], [-inf, -1e38, inf, inf],
             [0, -0.0, 0, 0], [-5, nan, -5, -4]]
    want = [1, 0, 0, 0, 0, 0, 2, 2, 0, 3]
    for width in (4, 5000):                                        # one split, several
        logits = torch.full((len(cases), width), -inf, device="cuda")
        at = [0, 1, width // 2, width - 1]
        for i, c in enumerate(cases):
            logits[i, at] = torch.tensor(c, dtype=torch.float32, device="cuda")
        expect = [at[w] for w in want]
        n = len(cases)
        # each row its own sequence: its id is the one kept
        tree = rt.TreeRows(torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"),
                           torch.zeros(n, 1, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int64, device="cuda"), n_rows=n)
        k = rt.tree_accept(tree, logits, torch.zeros(n, dtype=torch.int32, device="cuda"))
        assert k.ids.tolist() == expect and k.rows.tolist() == list(range(n)) and k.start.tolist() == list(range(n + 1))
        assert k.ids.tolist() == [int(rt.argmax(r.contiguous())) for r in logits]      # the rule of the greedy choice


def test_first_of_equal_children_and_wrong_words(torch, rt):
    """Two children with the right token: the first; words that name later rows or none are no parents."""
    logits = torch.zeros(6, 8, device="cuda")
    logits[:, 3] = 1
    tokens = torch.full((6,), 3, dtype=torch.int32, device="cuda")
    seen = [0b1, 0b111111, 0b111000, 0b000001, 0b1, 0b1001]        # 1: parent 0; 2: none; 3: 0; 4: 0; 5: 3
    tree = rt.TreeRows(torch.tensor([0, 6], dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda"),
                       torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor(seen, dtype=torch.int64, device="cuda"), n_rows=6)
    k = rt.tree_accept(tree, logits, tokens)
    assert k.start.tolist() == [0, 2] and k.rows.tolist()[:2] == [0, 1] and k.kv_len.tolist() == [6]
    tokens[1] = 2
    k = rt.tree_accept(tree, logits, tokens)
    assert k.start.tolist() == [0, 3] and k.rows.tolist()[:3] == [0, 3, 5]


def test_kv_len_of_the_tree_itself(torch, rt):
    tree, logits, parents, start, tokens = accept_case(torch, rt, [9, 0, 20], 300, seed=4)
    kept = rt.TreeKept(tree, kv_len=tree.kv_len)
    paths = check_acceptance(torch, rt, tree, logits, parents, start, tokens, kept)
    assert tree.kv_len.tolist() == [10 * (s + 1) + len(p) for s, p in enumerate(paths)]


def test_acceptance_of_bad_rows(torch, rt):
    """Too many rows, overlapping and falling ranges: nothing is written past the arrays, and it is flagged."""
    tree, logits, parents, start, tokens = accept_case(torch, rt, [30, 40], 300, seed=5)
    tok = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    tree.row_start.copy_(torch.tensor([0, 65, 70], dtype=torch.int32))
    k = rt.tree_accept(tree, logits, tok)
    assert k.start.tolist()[:2] == [0, 0] and k.kv_len.tolist()[0] == 10
    with pytest.raises(rt.B2Error, match="more drafted rows"):
        tree.check()
    n = 40
    tree = rt.TreeRows(torch.tensor([0, 3, 0] * 20, dtype=torch.int32, device="cuda"), torch.zeros(59, dtype=torch.int32, device="cuda"),
                       torch.zeros(59, 1, dtype=torch.int32, device="cuda"), torch.ones(5, dtype=torch.int64, device="cuda"), n_rows=5)
    arrays = torch.full((4, n + 60), -3, dtype=torch.int32, device="cuda")
    kept = rt.TreeKept(tree, arrays[0, :60], arrays[1, :59], arrays[2, :5], arrays[3, :5])
    rt.tree_accept(tree, logits[:5], tok[:5].contiguous(), kept)
    with pytest.raises(rt.B2Error, match="overlap"):
        tree.check()
    assert bool((arrays[0, 60:] == -3).all() & (arrays[1, 59:] == -3).all() & (arrays[2:, 5:] == -3).all())
    assert kept.start.amax() <= 5 and bool(((arrays[2, :5] >= -3) & (arrays[2, :5] < 5)).all())


@pytest.mark.parametrize("starts", [[0, 10, 5], [0, 10, 0], [0, 4, 10, 7], [0, 10, -3], [0, 10, 10, 2, 2]])
def test_ids_are_of_rows_whose_logits_were_looked_at(torch, rt, starts):
    """The last start lies below an earlier one: whatever the workspace held, an id is a row's own, and what is left of a
    path is its beginning."""
    import random
    n, vocab = 10, 5000
    g, rng = torch.Generator(device="cuda").manual_seed(sum(starts)), random.Random(len(starts))
    logits = torch.randn(n, vocab, device="cuda", generator=g)
    ids = logits.argmax(-1).tolist()
    i32 = dict(dtype=torch.int32, device="cuda")
    ends = [max(a, b) for a, b in zip(starts, starts[1:])]
    parents = [parents_of(rng, e - a, "chain") for a, e in zip(starts, ends) if a >= 0]
    seen, tokens = [1] * n, [0] * n
    for (a, e), p in zip(zip(starts, ends), parents):              # every draft is right: whole chains are accepted
        for j, word in enumerate(rt.tree_seen(p)):
            if a + j < n:
                seen[a + j], tokens[a + j] = word, ids[a + j - 1]
    ns = len(starts) - 1
    tree = rt.TreeRows(torch.tensor(starts, **i32), torch.full((ns,), 20, **i32), torch.zeros(ns, 1, **i32),
                       torch.tensor(seen, dtype=torch.int64, device="cuda"), n_rows=n)
    ws = rt.tree_accept_workspace(tree, vocab)
    for fill in (0x00, 0x5a, 0xff):
        ws.fill_(fill)
        kept = rt.TreeKept(tree)
        kept.rows.fill_(-7)
        kept.ids.fill_(-7)
        rt.tree_accept(tree, logits, torch.tensor(tokens, **i32), kept, workspace=ws)
        with pytest.raises(rt.B2Error, match="row_start below"):
            tree.check()
        last = max(starts[-1], 0)
        want = [list(range(a, min(e, last))) if a >= 0 else [] for a, e in zip(starts, ends)]
        flat = sum(want, [])
        total = len(flat)
        assert kept.start.tolist() == [sum(map(len, want[:s])) for s in range(ns + 1)]
        assert kept.kv_len.tolist() == [20 + len(w) for w in want]
        assert kept.rows.tolist() == flat + [-7] * (n - total) and kept.ids.tolist() == [ids[r] for r in flat] + [-7] * (n - total)


@pytest.mark.parametrize("n_seq,n_rows", [(0, 0), (0, 3), (1, 0), (3, 0), (700, 0)])
@pytest.mark.parametrize("own_lengths", [True, False])
def test_acceptance_of_no_rows(torch, rt, n_seq, n_rows, own_lengths):
    """Sums of nothing, and the lengths as they were."""
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = [5 + s for s in range(n_seq)]
    tree = rt.TreeRows(torch.zeros(n_seq + 1, **i32), torch.tensor(lens, **i32), torch.zeros(n_seq, 2, **i32),
                       torch.ones(n_rows, dtype=torch.int64, device="cuda"), n_rows=n_rows)
    kept = rt.TreeKept(tree, start=torch.full((n_seq + 1,), -7, **i32), kv_len=tree.kv_len if own_lengths else torch.full((n_seq,), -7, **i32))
    rt.tree_accept(tree, torch.randn(n_rows, 50, device="cuda"), torch.zeros(n_rows, **i32), kept)
    assert kept.start.tolist() == [0] * (n_seq + 1) and kept.kv_len.tolist() == lens and tree.kv_len.tolist() == lens
    tree.check()
    if n_seq:
        tree.row_start[0] = 2
        rt.tree_accept(tree, torch.randn(n_rows, 50, device="cuda"), torch.zeros(n_rows, **i32), kept)
        with pytest.raises(rt.B2Error, match="row_start below"):
            tree.check()


def test_captured_acceptance(torch, rt):
    tree, logits, parents, start, tokens = accept_case(torch, rt, [9, 12], 5000, seed=6)
    tok = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    kept, ws = rt.TreeKept(tree), rt.tree_accept_workspace(tree, 5000)
    rt.tree_accept(tree, logits, tok, kept, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.tree_accept(tree, logits, tok, kept, workspace=ws)
    for seed in (7, 8):
        _, l2, _, _, _ = accept_case(torch, rt, [9, 12], 5000, seed=seed)
        logits.copy_(l2)
        ids = logits.argmax(-1).tolist()
        t2 = [ids[a + up] if up >= 0 else 0 for a, p in zip(start, parents) for up in p]   # everything is right
        tok.copy_(torch.tensor(t2, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        top = logits.amax(-1, keepdim=True)
        first = torch.where(logits == top, torch.arange(5000, device="cuda"), 5000).amin(-1).tolist()
        paths = [accept_plain(p, t2[a:], first[a:]) for p, a in zip(parents, start)]
        n = sum(map(len, paths))
        assert kept.rows.tolist()[:n] == [a + i for p, a in zip(paths, start) for i in p] and kept.start.tolist()[-1] == n


# ------------------------------------------------------------------ appending what is kept
def table64(torch, n, d):
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    return torch.stack((ang.cos(), ang.sin()), -1).reshape(n, d).float()


def kept_case(torch, rt, counts, cached, KVH, dh, page, seed=0):
    """Two equal caches with room behind `cached` keys, and kept rows: counts[s] of each sequence, picked in no order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cap = -(-(max(cached) + 64) // page) * page
    pages = len(counts) * cap // page
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).reshape(len(counts), -1)
    n = sum(counts)
    src = n + 9
    pick = torch.randperm(src, device="cuda", generator=g)[:n].to(torch.int32)
    start = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    length = torch.tensor([c + k for c, k in zip(counts, cached)], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(src, KVH * dh + 4, device="cuda", generator=g)[:, :KVH * dh] for _ in range(2))
    caches = []
    codes = [torch.randint(-127, 128, (pages, KVH, page, dh), device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [0.005 + 0.02 * torch.rand(pages, KVH, page // 16, device="cuda", generator=g) for _ in range(2)]
    for _ in range(2):
        caches.append(rt.PagedKV(*(x.clone() for x in codes), *(x.clone() for x in scales)))
    seen = torch.ones(src, dtype=torch.int64, device="cuda")
    tree = rt.TreeRows(start, torch.tensor(cached, dtype=torch.int32, device="cuda"), table, seen, n_rows=src)
    rows = torch.full((src,), -1, dtype=torch.int32, device="cuda")
    rows[:n] = pick
    kept = rt.TreeKept(tree, start=start, kv_len=length, rows=rows)
    return caches, kept, k, v, pick


@pytest.mark.parametrize("dh", [16, 32, 64, 80, 128, 256])
@pytest.mark.parametrize("counts,cached", [([1], [0]), ([3], [15]), ([0, 17, 5, 1, 64], [3, 31, 16, 100, 7])])
@pytest.mark.parametrize("norm", [False, True])
def test_kept_rows_are_appended_as_the_same_rows_in_order(torch, rt, counts, cached, dh, norm):
    """Bit for bit what kv_append_i8 does with the rows gathered."""
    (a, b), kept, k, v, pick = kept_case(torch, rt, counts, cached, 3, dh, 32, seed=dh)
    table = table64(torch, 256, dh)
    gain = 1 + 0.1 * torch.randn(dh, device="cuda") if norm else None
    rt.kv_append_kept_i8(a, kept, k, v, table=table, k_gain=gain, eps=EPS)
    n = pick.shape[0]
    rows = rt.KVRows(kept.start, kept.kv_len, kept.tree.page_table, n_rows=n)
    rt.kv_append_i8(b, rows, k[pick.long()], v[pick.long()], table=table, k_gain=gain, eps=EPS)
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        assert torch.equal(x, y)
    a.check()


@pytest.mark.parametrize("eps", [EPS, 0.0])
def test_an_index_outside_the_rows_writes_zeros(torch, rt, eps):
    (a, b), kept, k, v, pick = kept_case(torch, rt, [7, 5], [20, 16], 2, 64, 16, seed=1)
    kept.rows[3], kept.rows[8] = -1, k.shape[0]
    gain = torch.ones(64, device="cuda")
    rt.kv_append_kept_i8(a, kept, k, v, k_gain=gain, eps=eps)
    with pytest.raises(rt.B2Error, match="row index"):
        a.check()
    kb, vb = k[pick.long()], v[pick.long()]
    kb[3], kb[8], vb[3], vb[8] = 0, 0, 0, 0
    rt.kv_append_i8(b, rt.KVRows(kept.start, kept.kv_len, kept.tree.page_table, n_rows=12), kb, vb, k_gain=gain, eps=EPS)
    assert torch.equal(a.v, b.v) and torch.equal(a.v_scale, b.v_scale)
    x, y = (rt.kv_read_i8(c, rt.KVRows(kept.start, kept.kv_len, kept.tree.page_table, n_rows=12))[0] for c in (a, b))
    assert not x[3].any() and not x[8].any() and bool(((x - y).abs() <= 1e-4).all()) == (eps == EPS) or eps == 0.0
    assert not x.isnan().any()


@pytest.mark.parametrize("eps", [EPS, 0.0])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_rows_of_a_bad_index_are_zeros_and_the_others_as_ever(torch, rt, eps, dh):
    """With and without an eps beneath the square root (a missing row has none of its own): beside an append of the same
    rows whose bad ones hold numbers, which share blocks with the others but not their norm; values bit for bit."""
    (a, b), kept, k, v, pick = kept_case(torch, rt, [7, 5, 16], [20, 16, 32], 2, dh, 16, seed=dh)
    bad = [3, 8]
    kept.rows[bad[0]], kept.rows[bad[1]] = -1, k.shape[0]
    gain = 1 + 0.1 * torch.randn(dh, device="cuda")
    rt.kv_append_kept_i8(a, kept, k, v, k_gain=gain, eps=eps)
    with pytest.raises(rt.B2Error, match="row index"):
        a.check()
    rows = rt.KVRows(kept.start, kept.kv_len, kept.tree.page_table, n_rows=28)
    kb, vb = k[pick.long()].clone(), v[pick.long()].clone()
    vb[bad] = 0
    kb[bad] = 1e-3                                                 # normed, elements of about the gain: never a block's largest
    rt.kv_append_i8(b, rows, kb, vb, k_gain=gain, eps=eps)
    assert torch.equal(a.v, b.v) and torch.equal(a.v_scale, b.v_scale)
    x, y = (rt.kv_read_i8(c, rows)[0] for c in (a, b))
    good = [i for i in range(28) if i not in bad]
    assert not x[bad].any() and bool(y[bad].any()) and not x.isnan().any()
    # blocks without a bad row: the same codes; with one: scales may differ if the bad row held the largest, which it does not
    assert torch.equal(x[good], y[good])


def test_kept_rows_past_the_capacity_or_the_table(torch, rt):
    (a, _), kept, k, v, _ = kept_case(torch, rt, [7], [90], 2, 64, 16, seed=2)
    before = a.k.clone()
    rt.kv_append_kept_i8(a, kept, k, v, table=table64(torch, 92, 64))       # positions 92 on have no rotation
    with pytest.raises(rt.B2Error, match="capacity"):
        a.check()
    page = int(kept.tree.page_table[0, 5])
    assert torch.equal(a.k[page, :, 12:], before[page, :, 12:]) and not torch.equal(a.k[page, :, 10:12], before[page, :, 10:12])
    kept.kv_len.fill_(1 << 20)
    rt.kv_append_kept_i8(a, kept, k, v)
    with pytest.raises(rt.B2Error, match="capacity"):
        a.check()


# ------------------------------------------------------------------ a verification step
def test_steps_of_a_served_batch(torch, rt, pkg):
    """Three steps of two sequences through the whole run: 4-bit products, norm and rotation, tree attention, products,
    acceptance, append, each captured once and replayed; beside it the same in 64 bits (over the cache's own values) and
    the cache that plain appends of the accepted rows make."""
    import random
    H, KVH, dh, d, V, page, n = 4, 2, 64, 256, 300, 16, 24
    rng, g = random.Random(0), torch.Generator(device="cuda").manual_seed(0)

    def weights(m, k):
        W, s = pkg.pack.quantize_groups_i4(torch.randn(m, k, device="cuda", generator=g).cpu().numpy() * k ** -0.5, 64)
        return torch.from_numpy(W).cuda(), torch.from_numpy(s).cuda()

    def wide(w, k):
        W, s = w
        c = torch.stack((W & 15, W >> 4), -1).flatten(1)[:, :k].to(torch.int32)
        return torch.where(c > 7, c - 16, c).double() * s.double().repeat_interleave(64, 1)[:, :k]

    w_qkv, w_o, w_head = weights((H + 2 * KVH) * dh, d), weights(d, H * dh), weights(V, d)
    embed = torch.randn(V, d, device="cuda", generator=g)
    table = table64(torch, 512, dh)
    lens = [37, 90]
    kv, twin = rt.PagedKV.empty(20, page, KVH, dh), rt.PagedKV.empty(20, page, KVH, dh)
    pages = torch.randperm(20, device="cuda", generator=g).to(torch.int32).reshape(2, 10)
    i32 = dict(dtype=torch.int32, device="cuda")
    length = torch.tensor(lens, **i32)
    first = rt.KVRows(torch.tensor([0, 37, 127], **i32), length.clone(), pages, n_rows=127)
    k0, v0 = (torch.randn(127, KVH * dh, device="cuda", generator=g) for _ in range(2))
    for c in (kv, twin):
        rt.kv_append_i8(c, first, k0, v0, table=table)
    start, seen = torch.tensor([0, 14, 24], **i32), torch.zeros(n, dtype=torch.int64, device="cuda")
    tokens, pos = torch.zeros(n, **i32), torch.zeros(n, **i32)
    tree = rt.TreeRows(start, length, pages, seen, n_rows=n, max_rows=14)
    kept = rt.TreeKept(tree, kv_len=length)
    ws = (rt.gemv_i4_groups_workspace(n, d), rt.attn_tree_workspace(kv, tree, H), rt.tree_accept_workspace(tree, V))
    state = {}

    def step():
        x = embed[tokens.long()]
        qkv = rt.gemv_i4_groups(*w_qkv, x, 64, workspace=ws[0])
        q, k, v = qkv[:, :H * dh], qkv[:, H * dh:(H + KVH) * dh], qkv[:, (H + KVH) * dh:]
        qr, kr = rt.qk_norm_rope(q, k, dh, pos=pos, table=table, q_scale=dh ** -0.5)
        att = rt.attn_tree_i8(kv, tree, qr, kr, v, workspace=ws[1])
        y = x + rt.gemv_i4_groups(*w_o, att, 64, workspace=ws[0])
        logits = rt.gemv_i4_groups(*w_head, y, 64, workspace=ws[0])
        rt.tree_accept(tree, logits, tokens, kept, workspace=ws[2])
        rt.kv_append_kept_i8(kv, kept, k, v, table=table)
        state.update(k=k, v=v, logits=logits, att=att)

    step()                                                         # warm-up on a tree of nothing but first rows
    torch.cuda.synchronize()
    length.copy_(torch.tensor(lens, **i32))
    for c in (kv, twin):
        for x in (c.k, c.v, c.k_scale, c.v_scale):
            x.zero_()
        rt.kv_append_i8(c, first, k0, v0, table=table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    length.copy_(torch.tensor(lens, **i32))
    now, known = list(lens), [5, 7]
    longest = 0
    for rnd in range(4):
        parents = [parents_of(rng, r, "tree") for r in (14, 10)]
        depth = []
        for s, p in enumerate(parents):
            dp = []
            for up in p:
                dp.append(dp[up] + 1 if up >= 0 else 0)
            depth += [now[s] + x for x in dp]
        pos.copy_(torch.tensor(depth, **i32))
        seen.copy_(torch.tensor(sum((rt.tree_seen(p) for p in parents), []), dtype=torch.int64))
        # drafts that are right: found by walking the model in 64 bits, row after row
        tok = [known[0]] + [rng.randrange(V) for _ in range(13)] + [known[1]] + [rng.randrange(V) for _ in range(9)]

        def model(tok):
            x = embed[torch.tensor(tok, device="cuda")].double()
            qkv = x @ wide(w_qkv, d).T
            t = table.double()[pos.long()]

            def turn(y, heads):
                y = y.reshape(n, heads, dh)
                a, b, c, s_ = y[..., 0::2], y[..., 1::2], t[:, None, 0::2], t[:, None, 1::2]
                return torch.stack((a * c - b * s_, a * s_ + b * c), -1).flatten(-2)
            q, k = turn(qkv[:, :H * dh], H) * dh ** -0.5, turn(qkv[:, H * dh:(H + KVH) * dh], KVH)
            v = qkv[:, (H + KVH) * dh:].reshape(n, KVH, dh)
            c = dict(kv=kv, tree=tree, table=pages, rows=[14, 10], cached=now, H=H, KVH=KVH, dh=dh, q=q.reshape(n, -1),
                     k=k.reshape(n, -1), v=v.reshape(n, -1))
            att, _ = attend64(torch, c)
            att = att.reshape(n, -1)
            return att, (x + att @ wide(w_o, H * dh).T) @ wide(w_head, d).T
        for s, a in ((0, 0), (1, 14)):
            for j, up in enumerate(parents[s]):
                if up >= 0 and rng.random() < 0.6:
                    tok[a + j] = int(model(tok)[1][a + up].argmax())
        att, logits = model(tok)
        tokens.copy_(torch.tensor(tok, **i32))
        graph.replay()
        torch.cuda.synchronize()
        # three products and an attention in f32 grade over values of order one
        assert float((state["att"].double() - att).abs().max()) < 1e-4 and float((state["logits"].double() - logits).abs().max()) < 1e-3
        top2 = logits.topk(2).values
        assert float((top2[:, 0] - top2[:, 1]).min()) > 0
        ids = state["logits"].argmax(-1).tolist()
        paths = [accept_plain(p, tok[a:], ids[a:]) for p, a in zip(parents, (0, 14))]
        longest = max(longest, *map(len, paths))
        flat = [a + i for p, a in zip(paths, (0, 14)) for i in p]
        now = [x + len(p) for x, p in zip(now, paths)]
        assert length.tolist() == now and kept.rows.tolist()[:len(flat)] == flat and kept.ids.tolist()[:len(flat)] == [ids[r] for r in flat]
        at = torch.tensor(flat, device="cuda")
        rt.kv_append_i8(twin, rt.KVRows(torch.tensor([0, len(paths[0]), len(flat)], **i32), torch.tensor(now, **i32), pages, n_rows=len(flat)),
                        state["k"][at], state["v"][at], table=table)
        for x, y in ((kv.k, twin.k), (kv.v, twin.v), (kv.k_scale, twin.k_scale), (kv.v_scale, twin.v_scale)):
            assert torch.equal(x, y)
        known = [ids[flat[len(paths[0]) - 1]], ids[flat[-1]]]
    assert longest > 2
    kv.check()
    tree.check()
