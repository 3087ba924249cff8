"""The paged 8-bit KV-cache operators as work to be measured: norms and rotation of queries and keys, appending to
the cache, reading rows back, and attention over it.

``run`` computes a case in its plain form (elementary torch operations) or, where ``own`` is true, through the calls
of ``runtime.py`` that a serving program makes: ``qk_norm_rope``, ``kv_append_i8``, ``kv_read_i8``, ``attn_paged_i8``.

A cache is a pool of pages. K and V are int8 codes [pages][kv_heads][page][d_head] with one f32 scale for each block of
16 tokens and head [pages][kv_heads][page / 16]; a sequence's keys lie in the pages that its row of the page table
lists. A call's rows are split over the sequences by ``row_start``; sequence s holds ``kv_len[s]`` keys with this call's
rows as the last of them.
"""
import math
import random

import torch

own = False

BLOCK = 16                       # tokens that share a scale
EPS = 1e-5
THETA = 10000.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a small grouped-query model between two matrix products: latency
        dict(name="norm-rope-1", op="norm_rope", n_seq=1, rows=1, ctx=1500, heads=32, kv_heads=4, d_head=64, page=16,
             norm=True, ragged=False, pad=0, mix=1),
        # a long prompt's queries and keys, an odd number of rows
        dict(name="norm-rope-8191", op="norm_rope", n_seq=1, rows=8191, ctx=0, heads=32, kv_heads=8, d_head=128,
             page=16, norm=True, ragged=False, pad=0, mix=2),
        # the newest token of one sequence: latency
        dict(name="append-1", op="append", n_seq=1, rows=1, ctx=639, heads=32, kv_heads=32, d_head=128, page=16,
             norm=False, ragged=False, pad=0, mix=3),
        # a decode step of 64 sequences of different lengths, blocks partly filled, in a padded batch
        dict(name="append-64", op="append", n_seq=64, rows=1, ctx=1151, heads=32, kv_heads=32, d_head=128, page=64,
             norm=True, ragged=True, pad=5, mix=4),
        # prompts of eight requests, each behind a cached prefix of its own length
        dict(name="append-prompts", op="append", n_seq=8, rows=1024, ctx=100, heads=32, kv_heads=8, d_head=128, page=32,
             norm=True, ragged=True, pad=0, mix=5),
        # a few rows read back, as a host does that moves one request
        dict(name="read-1", op="read", n_seq=1, rows=77, ctx=50, heads=32, kv_heads=4, d_head=64, page=16,
             norm=False, ragged=False, pad=0, mix=6),
        # whole caches of 16 sequences read back
        dict(name="read-16", op="read", n_seq=16, rows=1152, ctx=0, heads=32, kv_heads=32, d_head=128, page=64,
             norm=False, ragged=True, pad=0, mix=7),
        # one sequence's decode step: latency, the keys split over the GPU
        dict(name="attend-1", op="attend", n_seq=1, rows=1, ctx=639, heads=32, kv_heads=32, d_head=128, page=16,
             norm=False, ragged=False, pad=0, mix=8),
        # the batched decode step: 64 sequences, every head its own keys
        dict(name="attend-64", op="attend", n_seq=64, rows=1, ctx=1151, heads=32, kv_heads=32, d_head=128, page=64,
             norm=False, ragged=False, pad=0, mix=9),
        # few sequences with long caches and shared heads
        dict(name="attend-long", op="attend", n_seq=5, rows=1, ctx=40000, heads=32, kv_heads=4, d_head=64, page=128,
             norm=False, ragged=True, pad=0, mix=10),
        # a step of requests in different phases: pieces of prompts over caches, single tokens, in a padded batch
        dict(name="attend-mixed", op="attend", n_seq=12, rows=64, ctx=2000, heads=32, kv_heads=8, d_head=128, page=16,
             norm=False, ragged=True, pad=9, mix=11),
        # whole prompts
        dict(name="attend-prompts", op="attend", n_seq=4, rows=2047, ctx=0, heads=32, kv_heads=8, d_head=128, page=64,
             norm=False, ragged=False, pad=0, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("norm_rope", "append", "read", "attend", "attend"))
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (32, 4), (12, 12), (16, 2), (4, 2), (8, 1), (14, 7)))
        c = dict(op=op, n_seq=_log(rng, 1, 100), rows=1 if rng.random() < 0.4 else _log(rng, 2, 2500),
                 ctx=_log(rng, 1, 40000) - 1, heads=heads, kv_heads=kv_heads,
                 d_head=rng.choice((16, 64, 80, 96, 128, 128, 256)), page=rng.choice((16, 32, 64, 128)),
                 norm=rng.random() < 0.6, ragged=rng.random() < 0.7, pad=rng.choice((0, 0, 3, 17)), mix=rng.randrange(1 << 20))
        if op in ("norm_rope", "read"):
            c["ctx"] = min(c["ctx"], 2000)
        if op == "read":
            c.update(norm=False, pad=0)
        w, most = work(c), [work(x) for x in listed() if x["op"] == op]
        rows, keys = _sizes(c)
        full = len(rows) * max(rows) * max(keys) * heads * 4          # the plain form's scores, padded
        pool = 2 * len(rows) * max(keys) * kv_heads * c["d_head"] * 4  # and its gathered keys and values
        if (w["bytes"] <= max(x["bytes"] for x in most) and w["flops"] <= max(x["flops"] for x in most)
                and (op == "norm_rope" or pool <= 4e9) and (op != "attend" or full <= 2.5e9)):
            return c


def _sizes(case):
    """(rows, keys) of each sequence, from the case alone; ragged ones hold from none to all of the rows."""
    n, rows, ctx = case["n_seq"], case["rows"], case["ctx"]
    if not case["ragged"]:
        return [rows] * n, [rows + ctx] * n
    rng = random.Random(case["mix"])
    r = [rng.choice((1, rows, rng.randint(0, rows))) if case["op"] == "attend" else rng.randint((rows + 1) // 2, rows)
         for _ in range(n)]
    r[0] = rows
    return r, [x + rng.randint(ctx // 2, ctx) for x in r]


def work(case):
    rows, keys = _sizes(case)
    T, H, K, d = sum(rows), case["heads"], case["kv_heads"], case["d_head"]
    table = T * d * 4
    if case["op"] == "norm_rope":
        return {"bytes": 8 * T * (H + K) * d + table + 4 * T, "flops": 8 * T * (H + K) * d}
    if case["op"] == "append":
        # rows in, codes out, queries in and out; then the written blocks read back
        back = sum(r + (k - r) % BLOCK for r, k in zip(rows, keys))
        return {"bytes": T * K * d * (8 + 2) + 8 * T * H * d + table + back * K * d * 2 * 3 + back * K // 2,
                "flops": 8 * T * (H + 2 * K) * d + 2 * back * K * d}
    if case["op"] == "read":
        return {"bytes": T * K * d * 2 * 3 + T * K // 2, "flops": 2 * T * K * d}
    seen = sum(r * k - r * (r - 1) // 2 for r, k in zip(rows, keys))
    return {"bytes": sum(k for r, k in zip(rows, keys) if r) * K * (2 * d + 8 / BLOCK) + 8 * T * H * d,
            "flops": 4 * seen * H * d}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    op, H, K, d, page = case["op"], case["heads"], case["kv_heads"], case["d_head"], case["page"]
    rows, keys = _sizes(case)
    T, n = sum(rows), len(rows)
    s = dict(op=op, H=H, K=K, d=d, page=page, used=T, n_rows=T + case["pad"], max_rows=max(rows), max_keys=max(keys))
    row_start = [0]
    for r in rows:
        row_start.append(row_start[-1] + r)
    s["row_start"] = torch.tensor(row_start, dtype=torch.int32, device=dev)
    s["kv_len"] = torch.tensor(keys, dtype=torch.int32, device=dev)
    # the fused projection's output: queries, keys and values side by side
    qkv = normal(s["n_rows"], (H + 2 * K) * d)
    s["q"], s["k_new"], s["v_new"] = qkv[:, :H * d], qkv[:, H * d:(H + K) * d], qkv[:, (H + K) * d:]
    freq = THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
    angle = torch.arange(max(keys), device=dev, dtype=torch.float64)[:, None] * freq
    s["table"] = torch.stack((angle.cos(), angle.sin()), -1).reshape(max(keys), d).float()
    s["q_gain"] = 1 + 0.2 * normal(d) if case["norm"] else None
    s["k_gain"] = 1 + 0.2 * normal(d) if case["norm"] else None
    s["q_scale"] = d ** -0.5
    if op == "norm_rope":
        s["pos"] = torch.cat([torch.arange(k - r, k) for r, k in zip(rows, keys)]
                             + [torch.full((case["pad"],), -1)]).to(dev, torch.int32)
        s["q_out"] = torch.zeros(s["n_rows"], H * d, device=dev)
        s["k_out"] = torch.zeros(s["n_rows"], K * d, device=dev)
        return s
    # a pool with some pages to spare, handed out in no order
    need = [-(-k // page) for k in keys]
    n_pages, most = sum(need) + 3, max(need) + 1
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
        s[name + "_scale"] = (0.5 + torch.rand(n_pages, K, page // BLOCK, device=dev, generator=g)) / 36
    # queries as the attention takes them: rotated and scaled, some heads sharper than others
    if op == "attend":
        s["q"] = qkv[:, :H * d] * (d ** -0.5 * (0.5 + 2 * torch.rand(H, device=dev, generator=g))).repeat_interleave(d)
        s["out"] = torch.zeros(s["n_rows"], H * d, device=dev)
    if op == "append":
        s["q_out"] = torch.zeros(s["n_rows"], H * d, device=dev)
        # the blocks that the call writes to, whole, as rows to read back
        first = [k - r - (k - r) % BLOCK for r, k in zip(rows, keys)]
        back = [0]
        for f, k, r in zip(first, keys, rows):
            back.append(back[-1] + (k - f if r else 0))
        s["back_start"], s["back_rows"] = torch.tensor(back, dtype=torch.int32, device=dev), back[-1]
        s["live"] = torch.tensor([i for i, r in enumerate(rows) if r], device=dev)
    return s


# ------------------------------------------------------------------ plain forms
def _row_places(s, row_start, used):
    """(sequence, position, page) of each of the first `used` rows."""
    row = torch.arange(used, device=row_start.device)
    seq = torch.searchsorted(row_start[1:].long(), row, right=True)
    pos = s["kv_len"].long()[seq] - row_start.long()[seq + 1] + row
    return seq, pos, s["page_table"].long()[seq, pos // s["page"]]


def _normed_rotated(x, gain, table, dtype):
    """x [n][heads][d]: the norm of each head, then the rotation of neighbouring pairs by table [n][d]."""
    x = x.to(dtype)
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.to(dtype)
    pair, turn = x.unflatten(-1, (-1, 2)), table.to(dtype).unflatten(-1, (-1, 2))[:, None]
    a, b, c, t = pair[..., 0], pair[..., 1], turn[..., 0], turn[..., 1]
    return torch.stack((a * c - b * t, a * t + b * c), -1).flatten(-2)


def _plain_norm_rope(s):
    n, d = s["used"], s["d"]
    table = s["table"][s["pos"][:n].long()]
    q = _normed_rotated(s["q"][:n].unflatten(-1, (-1, d)), s["q_gain"], table, torch.float32) * s["q_scale"]
    k = _normed_rotated(s["k_new"][:n].unflatten(-1, (-1, d)), s["k_gain"], table, torch.float32)
    s["q_out"][:n] = q.flatten(1)
    s["k_out"][:n] = k.flatten(1)
    return s["q_out"], s["k_out"]


def _plain_write(s, name, x, seq, pos, page):
    """Rows x [n][kv_heads][d] (64 bits: codes lie next to borders) into the cache, each block's scale grown to hold
    its largest value and the rows that were there brought to the new scale."""
    codes = s[name].unflatten(2, (-1, BLOCK))                       # [pages][kv_heads][blocks][16][d]
    scale = s[name + "_scale"]
    blk, off = pos % s["page"] // BLOCK, pos % BLOCK
    cell = page * scale.shape[2] + blk                              # [n]
    cells, K = scale.shape[0] * scale.shape[2], x.shape[1]
    top = torch.zeros(cells, K, dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, cell[:, None].expand(-1, K), x.abs().amax(-1), "amax")
    # a block whose first token is in this call starts afresh
    fresh = torch.zeros(cells, dtype=torch.int64, device=x.device).scatter_reduce_(0, cell, (off == 0).long(), "amax")
    old = scale.transpose(1, 2).reshape(cells, K) * (1 - fresh)[:, None]
    new = torch.maximum(old, (top / 127).float())
    # only the block of a sequence's first row can hold older rows
    first = s["row_start"].long()[s["live"]]
    at = cell[first]
    ratio = torch.where(new[at] > 0, old[at] / new[at], 1.0).double()[:, :, None, None]
    there = codes[page[first], :, blk[first]].double()
    codes[page[first], :, blk[first]] = (there * ratio).round().to(torch.int8)
    mine = new[cell].double()[..., None]
    quotient = torch.where(mine > 0, x / mine, 0.0)
    codes[page, :, blk, off] = quotient.round().clamp(-127, 127).to(torch.int8)
    scale[page, :, blk] = new[cell]


def _plain_read(s, name, seq, pos, page):
    """[n][kv_heads][d] f32: the values that the codes stand for."""
    head = torch.arange(s["K"], device=pos.device)[None, :]
    off = (pos % s["page"])[:, None]
    return s[name][page[:, None], head, off].float() * s[name + "_scale"][page[:, None], head, off // BLOCK][..., None]


def _plain_append(s):
    n, d = s["used"], s["d"]
    seq, pos, page = _row_places(s, s["row_start"], n)
    table = s["table"][pos]
    q = _normed_rotated(s["q"][:n].unflatten(-1, (-1, d)), s["q_gain"], table, torch.float32) * s["q_scale"]
    s["q_out"][:n] = q.flatten(1)
    _plain_write(s, "k", _normed_rotated(s["k_new"][:n].unflatten(-1, (-1, d)), s["k_gain"], table, torch.float64),
                 seq, pos, page)
    _plain_write(s, "v", s["v_new"][:n].unflatten(-1, (-1, d)).double(), seq, pos, page)
    there = _row_places(s, s["back_start"], s["back_rows"])
    return (s["q_out"], *(_plain_read(s, x, *there).flatten(1).bfloat16() for x in ("k", "v")))


def _plain_attend(s):
    n, d, G = s["used"], s["d"], s["H"] // s["K"]
    dev = s["q"].device
    seqs, keys = s["kv_len"].shape[0], s["max_keys"]
    seq, pos, _ = _row_places(s, s["row_start"], n)
    at = torch.arange(n, device=dev) - s["row_start"].long()[seq]   # the row's number within its sequence
    q = torch.zeros(seqs, s["max_rows"], s["K"], G, d, device=dev)
    q[seq, at] = s["q"][:n].unflatten(-1, (s["K"], G, d))
    limit = torch.full((seqs, s["max_rows"]), -1, dtype=torch.long, device=dev)
    limit[seq, at] = pos                                            # the last key that the row sees
    j = torch.arange(keys, device=dev)
    held = j[None, :] < s["kv_len"][:, None]                        # [seqs][keys]
    page = torch.where(held, s["page_table"].long()[:, j // s["page"]], 0)
    head = torch.arange(s["K"], device=dev)[:, None, None]

    def values(name):                                               # [kv_heads][seqs][keys][d]
        off = j % s["page"]
        x = s[name][page, head, off].float()
        return x * torch.where(held, s[name + "_scale"][page, head, off // BLOCK], 0.0)[..., None]

    score = torch.einsum("sqhgd,hskd->shgqk", q, values("k"))
    score = torch.where(j <= limit[:, None, None, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.einsum("shgqk,hskd->sqhgd", p, values("v"))
    s["out"][:n] = out[seq, at].flatten(1)
    return s["out"]


# ------------------------------------------------------------------ the framework's calls
def _handles(s):
    """What a serving program keeps beside its tensors: the cache's and the plan's handles."""
    import importlib
    rt = importlib.import_module("aricode-ml_b200").runtime
    h = {"rt": rt}
    if s["op"] != "norm_rope":
        h["kv"] = rt.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
        plan = dict(kv_len=s["kv_len"], page_table=s["page_table"], max_keys=s["max_keys"])
        h["rows"] = rt.KVRows(s["row_start"], n_rows=s["n_rows"], max_rows=s["max_rows"], **plan)
        if s["op"] == "append":
            h["back"] = rt.KVRows(s["back_start"], n_rows=s["back_rows"], **plan)
        if s["op"] == "attend":
            h["workspace"] = rt.attn_paged_workspace(h["kv"], h["rows"], s["H"])
    return h


def run(state):
    s = state
    if not own:
        if s["op"] == "norm_rope":
            return _plain_norm_rope(s)
        if s["op"] == "append":
            return _plain_append(s)
        if s["op"] == "attend":
            return _plain_attend(s)
        there = _row_places(s, s["row_start"], s["used"])
        return tuple(_plain_read(s, x, *there).flatten(1).bfloat16() for x in ("k", "v"))
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    rt = h["rt"]
    if s["op"] == "norm_rope":
        return rt.qk_norm_rope(s["q"], s["k_new"], s["d"], pos=s["pos"], table=s["table"], q_gain=s["q_gain"],
                               k_gain=s["k_gain"], eps=EPS, q_scale=s["q_scale"], q_out=s["q_out"], k_out=s["k_out"])
    if s["op"] == "append":
        q = rt.kv_append_i8(h["kv"], h["rows"], s["k_new"], s["v_new"], table=s["table"], k_gain=s["k_gain"], eps=EPS,
                            q=s["q"], q_gain=s["q_gain"], q_scale=s["q_scale"], q_out=s["q_out"])
        return (q, *rt.kv_read_i8(h["kv"], h["back"], dtype=torch.bfloat16))
    if s["op"] == "attend":
        return rt.attn_paged_i8(h["kv"], h["rows"], s["q"], out=s["out"], workspace=h["workspace"])
    return rt.kv_read_i8(h["kv"], h["rows"], dtype=torch.bfloat16)


# ------------------------------------------------------------------ the definition in 64 bits
def _turn64(x, gain, table):
    """[n][heads][d] in 64 bits: normed if there is a gain, then each pair times the unit number of its angle."""
    x = x.double()
    if gain is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * gain.double()
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
    u = torch.view_as_complex(table.double().unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(z * u[:, None]).flatten(-2)


def _held64(s, name, i, count):
    """The first `count` values of sequence i in 64 bits: [count][kv_heads][d]."""
    pages = s["page_table"][i, :-(-count // s["page"])].long()
    x = s[name][pages].double() * s[name + "_scale"][pages].double().repeat_interleave(BLOCK, 2)[..., None]
    return x.permute(0, 2, 1, 3).reshape(-1, s["K"], s["d"])[:count]


def exact(case, seed):
    s = prepare(case, seed)
    rows, keys = _sizes(case)
    T, H, K, d, pad = s["used"], s["H"], s["K"], s["d"], case["pad"]
    split = [x.split(rows) for x in (s["q"][:T].unflatten(-1, (H, d)), s["k_new"][:T].unflatten(-1, (K, d)),
                                     s["v_new"][:T].unflatten(-1, (K, d)))]

    def whole(parts, width):
        return torch.cat([*(p.reshape(-1, width) for p in parts), torch.zeros(pad, width, dtype=torch.float64, device="cuda")])

    if case["op"] == "read":
        return tuple(torch.cat([_held64(s, x, i, k)[k - r:].flatten(1) for i, (r, k) in enumerate(zip(rows, keys))])
                     for x in ("k", "v"))
    if case["op"] == "attend":
        outs = []
        for i, (r, k) in enumerate(zip(rows, keys)):
            if r == 0:
                continue
            kk, vv = (_held64(s, x, i, k).repeat_interleave(H // K, 1).transpose(0, 1) for x in ("k", "v"))
            later = torch.ones(r, k, dtype=torch.bool, device="cuda").triu(k - r + 1)
            score = (split[0][i].double().transpose(0, 1) @ kk.transpose(1, 2)).masked_fill_(later, -math.inf)
            outs.append((torch.softmax(score, -1) @ vv).transpose(0, 1))
        return whole(outs, H * d)
    turned = []
    for which, gain in ((0, s["q_gain"]), (1, s["k_gain"])):
        turned.append([_turn64(split[which][i], gain, s["table"][k - r:k]) for i, (r, k) in enumerate(zip(rows, keys))])
    q = whole([x * s["q_scale"] for x in turned[0]], H * d)
    if case["op"] == "norm_rope":
        return q, whole(turned[1], K * d)
    values = []
    for name, new in (("k", turned[1]), ("v", [x.double() for x in split[2]])):
        out = []
        for i, (r, k) in enumerate(zip(rows, keys)):
            if r == 0:
                continue
            begin = (k - r) // BLOCK * BLOCK
            page = int(s["page_table"][i, begin // s["page"]])
            blk = begin % s["page"] // BLOCK
            for b in range(begin, k, BLOCK):
                lo, hi = max(b, k - r), min(b + BLOCK, k)
                x = new[i][lo - (k - r):hi - (k - r)]
                scale = (x.abs().amax((0, 2)) / 127).float()
                if lo > b:
                    was = s[name + "_scale"][page, :, blk]
                    scale = torch.maximum(scale, was)
                    old = s[name][page, :, blk * BLOCK:blk * BLOCK + lo - b].double().transpose(0, 1)
                    out.append((old * (was / scale).double()[None, :, None]).round() * scale.double()[None, :, None])
                unit = scale.double()[None, :, None]
                out.append((x / unit).round() * unit)
        values.append(torch.cat(out).flatten(1))
    return (q, *values)
