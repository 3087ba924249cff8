"""The operators of a step that verifies drafted tokens, as work to be measured: products with 4-bit weights that have
group scales, attention of a tree of drafted tokens over the paged 8-bit cache, accepting a path of the tree, and
appending the accepted rows to the cache.

``run`` computes a case in its plain form (elementary torch operations) or, where ``own`` is true, through the calls
of ``runtime.py`` that a serving program makes: ``gemv_i4_groups``, ``attn_tree_i8``, ``tree_accept``,
``kv_append_kept_i8`` (and ``kv_read_i8``, which reads the written blocks back).

Weights are signed 4-bit codes [m][ld bytes], two a byte with the even column in the low half, and a scale for each row
and group of columns. The cache is a pool of pages of int8 codes [pages][kv_heads][page][d_head] with one f32 scale for
each block of 16 tokens and head. Drafted rows are split over the sequences by ``row_start``; sequence s has
``kv_len[s]`` cached keys, and bit j of ``seen[i]`` says that row i also sees row j of its sequence. A row's parent is
the last row before it that it sees.
"""
import math
import random

import torch

own = False

BLOCK = 16                       # tokens that share a scale in the cache
EPS = 1e-5
THETA = 10000.0


# ------------------------------------------------------------------ cases
def listed():
    tree = dict(op="tree", ragged=False, pad=0)
    accept = dict(op="accept", ragged=True, pad=0)
    keep = dict(op="keep", ragged=True, pad=0)
    return [
        # one token through a square projection: latency
        dict(name="gemv-1", op="gemv", m=4096, n=4096, rows=1, group=128, bf16=True, bias=False, pad=0),
        # one token through the vocabulary projection: the largest matrix, read once
        dict(name="gemv-vocab", op="gemv", m=32000, n=4096, rows=1, group=64, bf16=True, bias=True, pad=0),
        # a small tree of drafts through the gate projection of a small model, slices of a wider buffer
        dict(name="gemv-13", op="gemv", m=5632, n=2048, rows=13, group=32, bf16=False, bias=False, pad=24),
        # four sequences with trees of sixteen drafts through the down projection
        dict(name="gemv-64", op="gemv", m=4096, n=11008, rows=64, group=128, bf16=True, bias=False, pad=0),
        # a short chain of drafts of one sequence: latency
        dict(tree, name="tree-1", n_seq=1, rows=5, ctx=639, heads=32, kv_heads=32, d_head=128, page=16, mix=1),
        # a batch of sequences with trees, every head its own keys
        dict(tree, name="tree-32", n_seq=32, rows=16, ctx=1152, heads=32, kv_heads=32, d_head=128, page=64, mix=2),
        # sequences of different lengths with trees of different sizes, shared heads, a padded batch
        dict(tree, name="tree-ragged", n_seq=16, rows=60, ctx=4000, heads=32, kv_heads=8, d_head=128, page=32, mix=3,
             ragged=True, pad=7),
        # few sequences with long caches and large trees
        dict(tree, name="tree-long", n_seq=2, rows=64, ctx=40000, heads=32, kv_heads=4, d_head=64, page=128, mix=4),
        # a chain of drafts of one sequence
        dict(accept, name="accept-1", n_seq=1, rows=8, ctx=639, vocab=32000, mix=5, ragged=False),
        # a batch, a vocabulary of odd size
        dict(accept, name="accept-48", n_seq=48, rows=25, ctx=1152, vocab=50257, mix=6, pad=3),
        # the accepted rows of one small tree
        dict(keep, name="keep-1", n_seq=1, rows=16, ctx=200, heads=32, kv_heads=4, d_head=64, page=16, mix=7,
             norm=False, ragged=False),
        # those of a batch, keys normed on the way
        dict(keep, name="keep-64", n_seq=64, rows=25, ctx=1152, heads=32, kv_heads=32, d_head=128, page=64, mix=8,
             norm=True, pad=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("gemv", "gemv", "tree", "tree", "accept", "keep"))
        if op == "gemv":
            c = dict(op=op, m=_log(rng, 1, 32000), n=_log(rng, 16, 16384), rows=1 if rng.random() < 0.3 else _log(rng, 2, 64),
                     group=rng.choice((32, 64, 128)), bf16=rng.random() < 0.5, bias=rng.random() < 0.4,
                     pad=rng.choice((0, 0, 4, 20)))
        else:
            c = dict(op=op, n_seq=_log(rng, 1, 64), rows=_log(rng, 1, 64), ctx=_log(rng, 1, 40000) - 1,
                     ragged=rng.random() < 0.7, pad=rng.choice((0, 0, 3, 17)), mix=rng.randrange(1 << 20))
            if op == "accept":
                c["vocab"] = rng.choice((256, 32000, 50257, _log(rng, 32, 130000)))
            else:
                c["heads"], c["kv_heads"] = rng.choice(((32, 32), (32, 8), (32, 4), (12, 12), (16, 2), (4, 2), (8, 1), (14, 7)))
                c.update(d_head=rng.choice((16, 64, 80, 96, 128, 128, 256)), page=rng.choice((16, 32, 64, 128)))
            if op == "keep":
                c.update(ctx=min(c["ctx"], 4000), norm=rng.random() < 0.6)
        w, most = work(c), [work(x) for x in listed() if x["op"] == op]
        if w["bytes"] > max(x["bytes"] for x in most) or w["flops"] > max(x["flops"] for x in most):
            continue
        if op in ("tree", "keep"):
            rows, ctx, _ = _plan(c)
            full = len(rows) * max(rows) * (max(ctx) + max(rows)) * c["heads"] * 4      # the plain form's scores, padded
            pool = 2 * len(rows) * (max(ctx) + 64) * c["kv_heads"] * c["d_head"] * 4    # and its gathered keys and values
            if pool > 4e9 or (op == "tree" and full > 2.5e9):
                continue
        return c


def _plan(case):
    """(rows, cached keys) of each sequence and the parents [sequence][row] of the drafted rows, from the case alone."""
    n, rows, ctx = case["n_seq"], case["rows"], case["ctx"]
    rng = random.Random(case["mix"])
    r, c = [rows] * n, [ctx] * n
    if case["ragged"]:
        r = [rows] + [rng.choice((1, rows, rng.randint(0, rows))) for _ in range(n - 1)]
        c = [rng.randint(ctx // 2, ctx) for _ in range(n)]
    # a chain with branches: each row follows the one before it, or any earlier one
    parents = [[-1] + [j - 1 if rng.random() < 0.5 else rng.randrange(j) for j in range(1, k)] if k else [] for k in r]
    return r, c, parents


def _accepted(case, parents):
    """The rows that a step keeps of each sequence: a path from its first row."""
    rng = random.Random(case["mix"] + 1)
    paths = []
    for p in parents:
        at = rng.randrange(len(p)) if p else -1
        path = []
        while at >= 0:
            path.append(at)
            at = p[at]
        paths.append(path[::-1])
    return paths


def work(case):
    if case["op"] == "gemv":
        m, n, T = case["m"], case["n"], case["rows"]
        return {"bytes": m * -(-n // 2) + m * -(-n // case["group"]) * (2 if case["bf16"] else 4) + 4 * T * (n + m)
                + (4 * m if case["bias"] else 0), "flops": 2 * m * n * T}
    rows, ctx, parents = _plan(case)
    T = sum(rows)
    if case["op"] == "accept":
        kept = sum(len(p) for p in _accepted(case, parents))
        return {"bytes": 4 * T * case["vocab"] + 12 * T + 12 * len(rows) + 8 * kept, "flops": T * case["vocab"]}
    H, K, d = case["heads"], case["kv_heads"], case["d_head"]
    if case["op"] == "keep":
        # the rows in, their codes out; then the written blocks read back
        paths = _accepted(case, parents)
        kept = sum(len(p) for p in paths)
        back = sum(len(p) + c % BLOCK for p, c in zip(paths, ctx))
        return {"bytes": kept * K * d * (8 + 2) + 4 * kept * (d + 1) + back * K * d * 2 * 3 + back * K // 2,
                "flops": 16 * kept * K * d + 2 * back * K * d}
    pairs = sum(r * c + sum(_depth(p)) for r, c, p in zip(rows, ctx, parents))
    return {"bytes": sum(c for r, c in zip(rows, ctx) if r) * K * (2 * d + 8 / BLOCK) + 8 * T * (H + K) * d + 8 * T,
            "flops": 4 * pairs * H * d}


def _depth(parents):
    """How many rows of its sequence each row sees, itself among them."""
    out = []
    for p in parents:
        out.append(1 + (out[p] if p >= 0 else 0))
    return out


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    if case["op"] == "gemv":
        m, n, T, group = case["m"], case["n"], case["rows"], case["group"]
        ld = (n + 31) // 32 * 16
        codes = torch.empty(m, 2 * ld, dtype=torch.int8, device=dev)
        for part in codes.view(-1).split(1 << 26):
            part.copy_((normal(part.numel()) * 2.7).round_().clamp_(-8, 7))
        W = (codes[:, 0::2] & 15 | codes[:, 1::2] << 4).view(torch.uint8)
        scale = (0.5 + uniform(m, -(-n // group))) * 0.007
        # hidden values of a normed row: a few channels are much larger than the others
        x = normal(T, n + case["pad"]) * (1 + 15 * (uniform(n + case["pad"]) < 0.004))
        return dict(op="gemv", m=m, n=n, group=group, W=W, scale=scale.bfloat16() if case["bf16"] else scale,
                    x=x[:, :n], bias=normal(m) if case["bias"] else None, y=torch.zeros(T, m, device=dev))
    op, (rows, ctx, parents) = case["op"], _plan(case)
    T, n = sum(rows), len(rows)
    s = dict(op=op, used=T, n_rows=T + case["pad"], max_rows=max(rows), max_keys=max(ctx))
    row_start, seen, depth, parent = [0], [], [], []
    for r, p in zip(rows, parents):
        see = []
        for j, up in enumerate(p):
            see.append((see[up] if up >= 0 else 0) | 1 << j)
            parent.append(row_start[-1] + up if up >= 0 else -1)
        row_start.append(row_start[-1] + r)
        seen += [x - (1 << 64) if x >> 63 else x for x in see]
        depth += _depth(p)
    s["row_start"] = torch.tensor(row_start, dtype=torch.int32, device=dev)
    s["kv_len"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
    s["seen"] = torch.tensor(seen + [0] * case["pad"], dtype=torch.int64, device=dev)
    if op == "accept":
        V = case["vocab"]
        # logits as bf16 products give them: whole steps, so that some rows have two largest ones
        s["logits"] = (normal(s["n_rows"], V) * 3).bfloat16().float()
        top = s["logits"].argmax(-1).to(torch.int32)
        # drafted tokens, most of them what the row before predicts
        up = torch.tensor(parent + [-1] * case["pad"], device=dev)
        guess = torch.randint(V, (s["n_rows"],), device=dev, generator=g, dtype=torch.int32)
        s["tokens"] = torch.where((up >= 0) & (uniform(s["n_rows"]) < 0.75), top[up.clamp(min=0)], guess)
        s["page_table"] = torch.zeros(n, 1, dtype=torch.int32, device=dev)
        s.update(_kept_buffers(n, s["n_rows"], dev))
        return s
    H, K, d, page = case["heads"], case["kv_heads"], case["d_head"], case["page"]
    s.update(H=H, K=K, d=d, page=page)
    # the fused projection's output: queries, keys and values side by side
    qkv = normal(s["n_rows"], (H + 2 * K) * d)
    s["q"], s["k_new"], s["v_new"] = qkv[:, :H * d], qkv[:, H * d:(H + K) * d], qkv[:, (H + K) * d:]
    # a pool with some pages to spare, handed out in no order; room for the accepted rows
    need = [-(-(c + 64) // page) for c in ctx]
    n_pages, most = sum(need) + 3, max(need)
    order = torch.randperm(n_pages, device=dev, generator=g).to(torch.int32)
    table = torch.full((n, most), -1, dtype=torch.int32, device=dev)
    where = torch.arange(most, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table[where] = order[:sum(need)]
    s["page_table"] = table
    for name in ("k", "v"):
        codes = torch.empty(n_pages, K, page, d, dtype=torch.int8, device=dev)
        for part in codes.view(-1).split(1 << 26):
            part.copy_((normal(part.numel()) * 36).round_().clamp_(-127, 127))
        s[name] = codes
        s[name + "_scale"] = (0.5 + uniform(n_pages, K, page // BLOCK)) / 36
    if op == "tree":
        # queries as the attention takes them: rotated and scaled, some heads sharper than others
        s["q"] = qkv[:, :H * d] * (d ** -0.5 * (0.5 + 2 * uniform(H))).repeat_interleave(d)
        s["out"] = torch.zeros(s["n_rows"], H * d, device=dev)
        return s
    paths = _accepted(case, parents)
    freq = THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
    angle = torch.arange(max(ctx) + 64, device=dev, dtype=torch.float64)[:, None] * freq
    s["table"] = torch.stack((angle.cos(), angle.sin()), -1).reshape(-1, d).float()
    s["k_gain"] = 1 + 0.2 * normal(d) if case["norm"] else None
    s.update(_kept_buffers(n, s["n_rows"], dev))
    start, back = [0], [0]
    for p, c in zip(paths, ctx):
        start.append(start[-1] + len(p))
        back.append(back[-1] + (len(p) + c % BLOCK if p else 0))
    s["kept_start"].copy_(torch.tensor(start, dtype=torch.int32))
    s["kept_len"].copy_(torch.tensor([c + len(p) for p, c in zip(paths, ctx)], dtype=torch.int32))
    s["kept"] = start[-1]
    s["kept_rows"][:s["kept"]] = torch.tensor([a + i for p, a in zip(paths, row_start) for i in p], dtype=torch.int32, device=dev)
    # the blocks that the call writes to, whole, as rows to read back
    s["back_start"], s["back_rows"] = torch.tensor(back, dtype=torch.int32, device=dev), back[-1]
    s["live"] = torch.tensor([i for i, p in enumerate(paths) if p], device=dev)
    return s


def _kept_buffers(n_seq, n_rows, dev):
    return {name: torch.full((size,), -1, dtype=torch.int32, device=dev)
            for name, size in (("kept_start", n_seq + 1), ("kept_len", n_seq), ("kept_rows", n_rows), ("kept_ids", n_rows))}


# ------------------------------------------------------------------ plain forms
def _plain_gemv(s):
    n, group = s["n"], s["group"]
    codes = torch.stack((s["W"] & 15, s["W"] >> 4), -1).flatten(1)[:, :n]
    w = ((codes ^ 8).float() - 8) * s["scale"].float().repeat_interleave(group, 1)[:, :n]
    y = s["x"] @ w.T
    s["y"].copy_(y if s["bias"] is None else y + s["bias"])
    return s["y"]


def _plain_tree(s):
    n, d, G, K = s["used"], s["d"], s["H"] // s["K"], s["K"]
    dev, seqs, keys, rows = s["q"].device, s["kv_len"].shape[0], s["max_keys"], s["max_rows"]
    row = torch.arange(n, device=dev)
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    at = row - s["row_start"].long()[seq]                           # the row's number within its sequence

    def padded(x, *shape):
        out = torch.zeros(seqs, rows, *shape, device=dev)
        out[seq, at] = x[:n].unflatten(-1, shape)
        return out

    q = padded(s["q"], K, G, d)
    see = torch.zeros(seqs, rows, dtype=torch.int64, device=dev)
    see[seq, at] = s["seen"][:n]
    # what each row sees: all cached keys, and the rows of its sequence that its bits name
    j = torch.arange(keys, device=dev)
    held = j < s["kv_len"][:, None]                                 # [seqs][keys]
    i = torch.arange(rows, device=dev)
    drafted = (see[:, :, None] >> i & 1).bool() & (i < (s["row_start"][1:] - s["row_start"][:-1])[:, None])[:, None]
    sees = torch.cat((held[:, None].expand(-1, rows, -1), drafted), -1)
    page = torch.where(held, s["page_table"].long()[:, j // s["page"]], 0)
    head = torch.arange(K, device=dev)[:, None, None]

    def values(name):                                               # [kv_heads][seqs][keys + rows][d]
        off = j % s["page"]
        x = s[name][page, head, off].float()
        x = x * torch.where(held, s[name + "_scale"][page, head, off // BLOCK], 0.0)[..., None]
        return torch.cat((x, padded(s[name + "_new"], K, d).permute(2, 0, 1, 3)), 2)

    score = torch.einsum("sqhgd,hskd->shgqk", q, values("k"))
    score = torch.where(sees[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.einsum("shgqk,hskd->sqhgd", p, values("v"))
    s["out"][:n] = out[seq, at].flatten(1)
    return s["out"]


def _plain_accept(s):
    n, dev, seqs, rows = s["used"], s["logits"].device, s["kv_len"].shape[0], s["max_rows"]
    logits = s["logits"][:n]
    V = logits.shape[1]
    top = logits.amax(-1, keepdim=True)
    ids = torch.where(logits == top, torch.arange(V, device=dev), V).amin(-1)
    row = torch.arange(n, device=dev)
    start = s["row_start"].long()
    seq = torch.searchsorted(start[1:], row, right=True)
    at = row - start[seq]
    # the parent: the last row before it that a row sees
    i = torch.arange(rows, device=dev)
    before = (s["seen"][:n, None] >> i & 1).bool() & (i < at[:, None])
    parent = torch.where(before, i, -1).amax(-1)
    follows = (parent >= 0) & (s["tokens"][:n].long() == ids[start[seq] + parent.clamp(min=0)])
    child = torch.full((seqs, rows), rows, device=dev)              # the first row that follows each one
    child.view(-1).scatter_reduce_(0, (seq * rows + parent.clamp(min=0))[follows], at[follows], "amin")
    # all sequences walk together: 0, its child, ...
    here = torch.where(start[1:] > start[:-1], 0, rows)
    path = []
    for _ in range(rows):
        path.append(here)
        here = torch.where(here < rows, child.gather(1, here.clamp(max=rows - 1)[:, None])[:, 0], rows)
    path = torch.stack(path, 1)                                     # [seqs][rows], `rows` where it has ended
    alive = path < rows
    count = alive.sum(1)
    s["kept_start"][0] = 0
    s["kept_start"][1:] = count.cumsum(0)
    s["kept_len"].copy_(s["kv_len"] + count)
    kept = (start[:-1, None] + path)[alive]
    s["kept_rows"][:kept.shape[0]] = kept.to(torch.int32)
    s["kept_ids"][:kept.shape[0]] = ids[kept].to(torch.int32)
    return s["kept_start"], s["kept_len"], s["kept_rows"], s["kept_ids"]


def _places(s, row_start, used):
    """(position, page) of each of the first `used` rows, which are the last of their sequence's kept_len keys."""
    row = torch.arange(used, device=row_start.device)
    seq = torch.searchsorted(row_start[1:].long(), row, right=True)
    pos = s["kept_len"].long()[seq] - row_start.long()[seq + 1] + row
    return pos, s["page_table"].long()[seq, pos // s["page"]]


def _plain_keep(s):
    n, d, K, page_size = s["kept"], s["d"], s["K"], s["page"]
    rows = s["kept_rows"][:n].long()
    pos, page = _places(s, s["kept_start"], n)
    # keys normed, then neighbouring pairs rotated (64 bits: codes lie next to borders)
    k = s["k_new"][rows].unflatten(-1, (K, d)).double()
    if s["k_gain"] is not None:
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_gain"].double()
    pair, turn = k.unflatten(-1, (-1, 2)), s["table"][pos].double().unflatten(-1, (-1, 2))[:, None]
    a, b, c, t = pair[..., 0], pair[..., 1], turn[..., 0], turn[..., 1]
    k = torch.stack((a * c - b * t, a * t + b * c), -1).flatten(-2)
    blk, off = pos % page_size // BLOCK, pos % BLOCK
    back, back_page = _places(s, s["back_start"], s["back_rows"])
    head = torch.arange(K, device=pos.device)[None, :]
    out = []
    for name, x in (("k", k), ("v", s["v_new"][rows].unflatten(-1, (K, d)).double())):
        codes, scale = s[name].unflatten(2, (-1, BLOCK)), s[name + "_scale"]
        blocks = scale.shape[2]
        cell = page * blocks + blk
        top = torch.zeros(scale.shape[0] * blocks, K, dtype=torch.float64, device=pos.device)
        top.scatter_reduce_(0, cell[:, None].expand(-1, K), x.abs().amax(-1), "amax")
        # a block whose first token is in this call starts afresh, the others' scales grow
        fresh = torch.zeros(top.shape[0], dtype=torch.int64, device=pos.device).scatter_reduce_(0, cell, (off == 0).long(), "amax")
        old = scale.transpose(1, 2).reshape(-1, K) * (1 - fresh)[:, None]
        new = torch.maximum(old, (top / 127).float())
        # only the block of a sequence's first row can hold older rows: to the new scale
        first = s["kept_start"].long()[s["live"]]
        was = cell[first]
        ratio = torch.where(new[was] > 0, old[was] / new[was], 1.0).double()[:, :, None, None]
        there = codes[page[first], :, blk[first]].double()
        codes[page[first], :, blk[first]] = (there * ratio).round().to(torch.int8)
        mine = new[cell].double()[..., None]
        codes[page, :, blk, off] = torch.where(mine > 0, x / mine, 0.0).round().clamp(-127, 127).to(torch.int8)
        scale[page, :, blk] = new[cell]
        at = (back % page_size)[:, None]
        value = s[name][back_page[:, None], head, at].float() * scale[back_page[:, None], head, at // BLOCK][..., None]
        out.append(value.flatten(1).bfloat16())
    return tuple(out)


# ------------------------------------------------------------------ the framework's calls
def _handles(s):
    """What a serving program keeps beside its tensors: the cache's and the plan's handles, workspaces."""
    import importlib
    rt = importlib.import_module("aricode-ml_b200").runtime
    h = {"rt": rt}
    if s["op"] == "gemv":
        h["workspace"] = rt.gemv_i4_groups_workspace(s["x"].shape[0], s["n"], device=s["x"].device)
        return h
    h["tree"] = rt.TreeRows(s["row_start"], s["kv_len"], s["page_table"], s["seen"], n_rows=s["n_rows"],
                            max_keys=s["max_keys"], max_rows=s["max_rows"])
    if s["op"] != "accept":
        h["kv"] = rt.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "tree":
        h["workspace"] = rt.attn_tree_workspace(h["kv"], h["tree"], s["H"])
        return h
    h["kept"] = rt.TreeKept(h["tree"], s["kept_start"], s["kept_len"], s["kept_rows"], s["kept_ids"])
    if s["op"] == "accept":
        h["workspace"] = rt.tree_accept_workspace(h["tree"], s["logits"].shape[1])
    else:
        h["back"] = rt.KVRows(s["back_start"], s["kept_len"], s["page_table"], n_rows=s["back_rows"])
    return h


def run(state):
    s = state
    if not own:
        return {"gemv": _plain_gemv, "tree": _plain_tree, "accept": _plain_accept, "keep": _plain_keep}[s["op"]](s)
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    rt = h["rt"]
    if s["op"] == "gemv":
        return rt.gemv_i4_groups(s["W"], s["scale"], s["x"], s["group"], bias=s["bias"], y=s["y"], workspace=h["workspace"])
    if s["op"] == "tree":
        return rt.attn_tree_i8(h["kv"], h["tree"], s["q"], s["k_new"], s["v_new"], out=s["out"], workspace=h["workspace"])
    if s["op"] == "accept":
        kept = rt.tree_accept(h["tree"], s["logits"], s["tokens"], h["kept"], workspace=h["workspace"])
        return kept.start, kept.kv_len, kept.rows, kept.ids
    rt.kv_append_kept_i8(h["kv"], h["kept"], s["k_new"], s["v_new"], table=s["table"], k_gain=s["k_gain"], eps=EPS)
    return rt.kv_read_i8(h["kv"], h["back"], dtype=torch.bfloat16)


# ------------------------------------------------------------------ the definition in 64 bits
def _held64(s, name, i, count):
    """The first `count` cached values of sequence i in 64 bits: [count][kv_heads][d]."""
    pages = s["page_table"][i, :-(-count // s["page"])].long()
    x = s[name][pages].double() * s[name + "_scale"][pages].double().repeat_interleave(BLOCK, 2)[..., None]
    return x.permute(0, 2, 1, 3).reshape(-1, s["K"], s["d"])[:count]


def exact(case, seed):
    if case["op"] == "accept":       # whole numbers alone
        return None
    s = prepare(case, seed)
    if case["op"] == "gemv":
        n, group, x = case["n"], case["group"], s["x"].double()
        y = torch.zeros(x.shape[0], case["m"], dtype=torch.float64, device="cuda")
        for g in range(0, n, group):
            b = s["W"][:, g // 2:(min(g + group, n) + 1) // 2].to(torch.int64)
            c = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.float64, device="cuda")
            for half in (0, 1):
                nibble = b >> 4 * half & 15
                c[:, half::2] = torch.where(nibble > 7, nibble - 16, nibble).double()
            cols = min(group, n - g)
            y += (x[:, g:g + cols] @ c[:, :cols].T) * s["scale"][:, g // group].double()
        return y if s["bias"] is None else y + s["bias"].double()
    rows, ctx, parents = _plan(case)
    T, K, d, H = s["used"], s["K"], s["d"], s["H"]
    k_new, v_new = (s[x][:T].unflatten(-1, (K, d)).double().split(rows) for x in ("k_new", "v_new"))
    if case["op"] == "tree":
        outs = []
        for i, (r, c, up) in enumerate(zip(rows, ctx, parents)):
            if r == 0:
                continue
            kk, vv = (torch.cat((_held64(s, x, i, c), new[i])).repeat_interleave(H // K, 1).transpose(0, 1)
                      for x, new in (("k", k_new), ("v", v_new)))
            hidden = torch.ones(r, r, dtype=torch.bool)
            for j in range(r):
                at = j
                while at >= 0:
                    hidden[j, at] = False
                    at = up[at]
            hidden = torch.cat((torch.zeros(r, c, dtype=torch.bool), hidden), 1).cuda()
            a = sum(rows[:i])
            q = s["q"][a:a + r].unflatten(-1, (H, d)).double().transpose(0, 1)
            outs.append((torch.softmax((q @ kk.transpose(1, 2)).masked_fill_(hidden, -math.inf), -1) @ vv).transpose(0, 1))
        return torch.cat([*(o.reshape(-1, H * d) for o in outs), torch.zeros(case["pad"], H * d, dtype=torch.float64, device="cuda")])
    values = {"k": [], "v": []}
    for i, (path, c) in enumerate(zip(_accepted(case, parents), ctx)):
        if not path:
            continue
        k = k_new[i][path]
        if s["k_gain"] is not None:
            k = k * (k.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * s["k_gain"].double()
        # each pair times the unit number of its angle
        unit = torch.view_as_complex(s["table"][c:c + len(path)].double().unflatten(-1, (-1, 2)).contiguous())
        k = torch.view_as_real(torch.view_as_complex(k.unflatten(-1, (-1, 2)).contiguous()) * unit[:, None]).flatten(-2)
        for name, new in (("k", k), ("v", v_new[i][path])):
            for b in range(c // BLOCK * BLOCK, c + len(path), BLOCK):
                x = new[max(b - c, 0):b + BLOCK - c]
                step = (x.abs().amax((0, 2)) / 127).float()
                if b < c:
                    page, blk, held = int(s["page_table"][i, b // s["page"]]), b % s["page"] // BLOCK, c - b
                    was = s[name + "_scale"][page, :, blk]
                    step = torch.maximum(step, was)
                    old = s[name][page, :, blk * BLOCK:blk * BLOCK + held].double().transpose(0, 1)
                    values[name].append((old * (was / step).double()[None, :, None]).round() * step.double()[None, :, None])
                values[name].append((x / step.double()[None, :, None]).round() * step.double()[None, :, None])
    return tuple(torch.cat(values[x]).flatten(1) for x in ("k", "v"))
