"""The paged serving operators, case by case: append, attention, shared-prefix attention, compaction.

One decoding step of a server that keeps its keys and values in pages: the fused projection's rows are
normalised, rotated and appended to the pages; every request's rows attend to its pages (causally, or
through the ancestor bits of a draft tree); requests with a common prompt read that prompt's pages once
for all of them; after verification the accepted rows move together.

``run`` computes a case in elementary torch operations, or (``own``) through ``woodcock_b200.ops``.

Layout: pages [pages][kv_heads][page_size][head_dim]; ``page_table`` int32 [B][max_pages]; ``kv_lens``
int32 [B] counts a request's keys, its new rows included; request b's new rows are
``q_offsets[b] .. q_offsets[b + 1]`` of q.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BASE = 1e6  # rotation base of the Qwen3 configurations
EPS = 1e-6


# ---------------------------------------------------------------------------- the cases


def listed():
    tall = {"heads": 16, "kv_heads": 8, "head_dim": 128}   # the 1.7B layout
    wide = {"heads": 32, "kv_heads": 8, "head_dim": 128}   # the 4B layout
    tiny = {"heads": 4, "kv_heads": 2, "head_dim": 64}     # the tiny fp32 model
    return [
        # 64 requests decode one token each; the projection GEMM leaves fp32 rows
        {"name": "append decode 64", "op": "append", **tall, "dtype": "bf16", "src": "fp32", "requests": 64, "rows": 1,
         "ragged": False, "len": 2049, "page": 16, "far": 0},
        # prompts of unequal length arrive together, far into a long session
        {"name": "append prompts", "op": "append", **wide, "dtype": "bf16", "src": "bf16", "requests": 5, "rows": 4099,
         "ragged": True, "len": 4400, "page": 64, "far": 1000003},
        # one request, one token: the latency of an interactive session
        {"name": "decode 1", "op": "attention", **tall, "dtype": "bf16", "requests": 1, "rows": 1, "ragged": False,
         "mask": "causal", "len": 513, "page": 16},
        # 64 requests of very unequal length, one token each, an idle slot among them
        {"name": "decode 64 ragged", "op": "attention", **wide, "dtype": "bf16", "requests": 64, "rows": 1,
         "ragged": True, "mask": "causal", "len": 12289, "page": 16},
        # the batched tree verification: 64 requests, 32 nodes each
        {"name": "tree verify 64x32", "op": "attention", **tall, "dtype": "bf16", "requests": 64, "rows": 32,
         "ragged": False, "mask": "tree", "len": 4128, "page": 64},
        # a prompt pass over prompts of unequal length
        {"name": "prompts ragged", "op": "attention", **wide, "dtype": "bf16", "requests": 4, "rows": 4096,
         "ragged": True, "mask": "causal", "len": 4096, "page": 64},
        # the fp32 model's chain verification
        {"name": "verify fp32", "op": "attention", **tiny, "dtype": "fp32", "requests": 8, "rows": 5, "ragged": False,
         "mask": "causal", "len": 600, "page": 16},
        # eight chains of five rows under one system prompt
        {"name": "prefix 8x5", "op": "prefix", **tall, "dtype": "bf16", "groups": 1, "requests": 8, "rows": 5,
         "ragged": False, "mask": "causal", "prefix": 1001, "len": 77, "page": 16},
        # many samples of a few long prompts, one token each
        {"name": "prefix 4 groups x 32", "op": "prefix", **wide, "dtype": "bf16", "groups": 4, "requests": 32,
         "rows": 1, "ragged": True, "mask": "causal", "prefix": 8191, "len": 1030, "page": 64},
        # tree verification of 64 requests under one long document
        {"name": "prefix tree 64x32", "op": "prefix", **tall, "dtype": "bf16", "groups": 1, "requests": 64, "rows": 32,
         "ragged": True, "mask": "tree", "prefix": 16384, "len": 512, "page": 64},
        # one request's accepted path after a tree of 16 nodes, every layer
        {"name": "compact 1", "op": "compact", "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "layers": 28,
         "requests": 1, "rows": 16, "accepted": 5, "len": 545, "page": 16},
        # the accepted paths of 64 requests after trees of 32 nodes, every layer
        {"name": "compact 64", "op": "compact", "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "layers": 28,
         "requests": 64, "rows": 32, "accepted": 5, "len": 128, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    ceiling = max(_cost(c) for c in listed())
    # a few rejections at most: each redraw shrinks the ranges' upper ends
    for shrink in range(12):
        c = _drawn(rng, 0.75 ** shrink)
        if _cost(c) <= ceiling:
            return c
    return {k: v for k, v in listed()[2].items() if k != "name"} | {"len": rng.randrange(2, 4000)}


def _drawn(rng, s):
    heads, kv = rng.choice([(16, 8), (32, 8), (4, 2), (8, 8), (8, 1), (40, 8), (6, 2)])
    c = {"op": rng.choice(["append", "attention", "attention", "prefix", "compact"]), "heads": heads, "kv_heads": kv,
         "head_dim": rng.choice([64, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "bf16", "fp32"]),
         "page": rng.choice([16, 32, 64, 128])}
    small = c["dtype"] == "fp32"

    def upto(lo, hi):
        return _log_int(rng, lo, max(lo, int(hi * s)))

    if c["op"] == "append":
        c |= {"src": rng.choice(["bf16", "fp32"]), "requests": upto(1, 128), "ragged": rng.random() < 0.5,
              "far": rng.choice([0, 0, 70001, 900007])}
        c["rows"] = upto(1, max(1, (2000 if small else 12000) // c["requests"]))
        c["len"] = c["rows"] + rng.randrange(0, 500)
    elif c["op"] == "compact":
        c |= {"layers": upto(1, 36), "requests": upto(1, 64), "rows": rng.randrange(2, 64)}
        c["accepted"] = rng.randrange(1, min(9, c["rows"] + 1))
        c["len"] = c["rows"] + rng.randrange(0, 200)
        del c["heads"]
    else:
        kind = rng.choice(["decode", "verify", "prompt"])
        c |= {"mask": "causal", "ragged": rng.random() < 0.5}
        if kind == "decode":
            c |= {"requests": upto(1, 96), "rows": 1}
            c["len"] = upto(1, (40000 if small else 300000) // c["requests"])
        elif kind == "verify":
            c |= {"requests": upto(1, 64), "rows": rng.randrange(2, 49), "mask": rng.choice(["tree", "causal"])}
            c["len"] = c["rows"] + upto(1, (20000 if small else 200000) // c["requests"])
        else:
            c |= {"requests": upto(1, 4), "rows": upto(65, 600 if small else 3000)}
            c["len"] = c["rows"] + rng.choice([0, 0, rng.randrange(0, 2000)])
        if c["op"] == "prefix":
            c["groups"] = upto(1, min(4, c["requests"]))
            c["requests"] = -(-c["requests"] // c["groups"])
            c["len"] = min(c["len"], c["rows"] + 1500)
            c["prefix"] = upto(1, 2000 if small else 12000)
    return c


# ---------------------------------------------------------------------------- sizes


def _rows_of(case):
    """New rows of each request: all alike, or from one up to ``rows``."""
    B, n = _requests(case), case["rows"]
    if not case.get("ragged") or n == 1:
        return [n] * B
    return [max(1, n if i == 0 else int(n * ((i * 0.6180339887) % 1.0))) for i in range(B)]


def _lens_of(case):
    """Keys of each request, its new rows included. Ragged: spread from short to ``len``; from three
    requests on, the last of a one-row batch is an idle slot (no keys)."""
    B, n = _requests(case), case["len"]
    rows = _rows_of(case)
    if not case.get("ragged"):
        return [max(n, r) for r in rows]
    lens = [max(r, n if i == 0 else int(n * ((i * 0.7548776662) % 1.0))) for i, r in enumerate(rows)]
    if case["op"] == "attention" and case["rows"] == 1 and B >= 3:
        lens[-1] = 0
    return lens


def _requests(case):
    return case["requests"] * case.get("groups", 1)


def _visible(case):
    """Sum over all query rows of the keys that each sees, the prefix not counted."""
    total = 0
    for r, n in zip(_rows_of(case), _lens_of(case)):
        if n == 0:
            continue
        total += r * (n - r) + (r * (r + 1) // 2 if case["mask"] == "causal" else r * min(r, 6))
    return total


def work(case):
    D, Hk = case["head_dim"], case["kv_heads"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "compact":
        # the first accepted row stays where it is, the others move: read and written once, K and V
        moved = (case["accepted"] - 1) * case["requests"] * case["layers"] * Hk * D * 2
        return {"bytes": max(2 * moved * e, 8 * case["requests"]), "flops": 0}
    H = case["heads"]
    T = sum(_rows_of(case))
    if case["op"] == "append":
        es = 2 if case["src"] == "bf16" else 4
        values = T * (H + 2 * Hk) * D
        return {"bytes": values * (es + e), "flops": 10 * values}
    keys, seen = sum(_lens_of(case)), _visible(case)
    if case["op"] == "prefix":
        keys += case["groups"] * case["prefix"]
        seen += T * case["prefix"]
    return {"bytes": (2 * keys * Hk + 2 * T * H) * D * e, "flops": 4 * seen * H * D}


def _cost(case):
    w = work(case)
    # fp32 products run without the matrix units
    return max(w["bytes"] / 6.4e12, w["flops"] / (1.6e15 if case["dtype"] == "bf16" else 4e13))


# ---------------------------------------------------------------------------- inputs


def _table(gen, lens, page, width=None, first=0):
    """A page table whose pages are scattered over the pool. Pages past a request's length are shared
    with nobody either: they are just not read. Returns (table, number of pages)."""
    width = width or max(1, max(-(-n // page) for n in lens))
    order = torch.randperm(len(lens) * width, generator=gen, device="cuda")
    return (first + order.reshape(len(lens), width)).to(torch.int32), first + len(lens) * width


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return _ints(out)


def _tree_bits(gen, rows, width):
    """Ancestor bits (itself included) of random draft trees: node 0 the root, node i's parent a node
    before it, more often a late one. int64 [sum(rows)]."""
    B = len(rows)
    u = torch.rand((B, width), generator=gen, device="cuda")
    bits = torch.zeros((B, width), dtype=torch.int64, device="cuda")
    bits[:, 0] = 1
    for i in range(1, width):
        parent = (i * u[:, i].sqrt()).long().clamp_(max=i - 1)
        bits[:, i] = bits.gather(1, parent[:, None])[:, 0] | (1 << i)
    keep = torch.arange(width, device="cuda")[None] < _ints(rows)[:, None]
    return bits[keep]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    dt = DTYPES[case["dtype"]]
    Hk, D, page = case["kv_heads"], case["head_dim"], case["page"]
    s = {"case": dict(case)}
    if case["op"] == "compact":
        B, n, a, L = case["requests"], case["rows"], case["accepted"], case["layers"]
        starts = [max(0, case["len"] - n - 7 * i % 61) for i in range(B)]
        table, pages = _table(gen, [x + n for x in starts], page)
        s |= {"k": torch.empty((L, pages, Hk, page, D), dtype=dt, device="cuda").normal_(generator=gen),
              "v": torch.empty((L, pages, Hk, page, D), dtype=dt, device="cuda").normal_(generator=gen),
              "table": table, "starts": _ints(starts)}
        # the path root -> ... of distinct nodes; nodes past the first come from the tree's later levels
        # (number a or later where there are enough of them), as breadth-first numbering gives
        later = max(a, 1) if n - a >= a - 1 else 1
        picks = torch.rand((B, n - later), generator=gen, device="cuda").argsort(1)[:, : a - 1].sort(1).values + later
        keep = torch.cat([torch.zeros((B, 1), dtype=torch.int64, device="cuda"), picks], 1) if a > 1 else \
            torch.zeros((B, 1), dtype=torch.int64, device="cuda")
        if later == 1:  # too few nodes to come from: the path is the chain itself
            keep = torch.arange(a, device="cuda").expand(B, a)
        s |= {"keep": keep.to(torch.int32).contiguous(), "n_keep": _ints([a] * B)}
        return s

    H = case["heads"]
    rows, lens = _rows_of(case), _lens_of(case)
    T = sum(rows)
    G = case.get("groups", 0)
    s["lens"] = _ints(lens)
    s["offsets"] = _offsets(rows) if case.get("ragged") else None
    s["table"], pages = _table(gen, lens, page)
    if case["op"] == "prefix":
        s["prefix_lens"] = _ints([case["prefix"]] * G)
        s["prefix_table"], pages = _table(gen, [case["prefix"]] * G, page, first=pages)
        s["groups"] = _offsets([case["requests"]] * G)
    if case["op"] == "append":
        # the fused projection's output: q | k | v side by side
        qkv = randn(T, (H + 2 * Hk) * D, dtype=DTYPES[case["src"]])
        s["q"] = qkv[:, : H * D].view(T, H, D)
        s["kn"] = qkv[:, H * D: (H + Hk) * D].view(T, Hk, D)
        s["vn"] = qkv[:, (H + Hk) * D:].view(T, Hk, D)
        s["q_norm"] = 1 + randn(D, scale=0.1)
        s["k_norm"] = 1 + randn(D, scale=0.1)
        s["k"] = torch.zeros((pages, Hk, page, D), dtype=dt, device="cuda")
        s["v"] = torch.zeros((pages, Hk, page, D), dtype=dt, device="cuda")
        # positions: the slot, moved by what earlier parts of the session took
        start = s["lens"] - _ints(rows)
        within = torch.cat([torch.arange(r, device="cuda", dtype=torch.int32) for r in rows])
        which = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), _ints(rows).long(), output_size=T)
        s["positions"] = (start[which] + within + case["far"]).to(torch.int32)
        return s
    # normalised keys, queries somewhat longer, so that some keys stand out
    s["q"] = randn(T, H, D, dtype=dt, scale=1.5)
    s["k"] = torch.empty((pages, Hk, page, D), dtype=dt, device="cuda").normal_(generator=gen)
    s["v"] = torch.empty((pages, Hk, page, D), dtype=dt, device="cuda").normal_(generator=gen)
    s["bits"] = _tree_bits(gen, rows, max(rows)) if case["mask"] == "tree" else None
    return s


# ---------------------------------------------------------------------------- the plain forms


def _row_ends(T, B, offsets):
    return torch.arange(0, T + 1, T // B, device="cuda") if offsets is None else offsets.long()


def _padded(o, most):
    """Index [B][most] of every request's rows, and which of them exist."""
    i = torch.arange(most, device="cuda")
    real = i[None] < (o[1:] - o[:-1])[:, None]
    return torch.where(real, o[:-1, None] + i[None], 0), real


def _rows_from_pages(pages, table):
    """[B][Hk][table width * page][D] in 32 bits."""
    g = pages[table.long()]  # [B][width][Hk][page][D]
    B, W, Hk, ps, D = g.shape
    return g.permute(0, 2, 1, 3, 4).reshape(B, Hk, W * ps, D).float()


def _attend(q, k, v, sees):
    """q [B][L][H][D], k / v [B][Hk][N][D], sees [B][L][N] -> [B][L][H][D]; rows that see nothing give 0."""
    B, L, H, D = q.shape
    Hk = k.shape[1]
    rep = H // Hk
    qh = q.float().view(B, L, Hk, rep, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, rep * L, D)
    z = (qh @ k.transpose(2, 3)).view(B, Hk, rep, L, -1) * D ** -0.5
    z = z.masked_fill_(~sees[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    e = (z - torch.where(top.isinf(), 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, Hk, rep * L, -1) @ v).view(B, Hk, rep, L, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, L, H, D)


def _sees(lens, rows_of, i, N, bits):
    """[B][L][N]: which of a request's N key slots its row i sees."""
    n = torch.arange(N, device="cuda")[None, None]
    first = (lens.long() - rows_of)[:, None, None]  # slot of the request's row 0
    inside = n < lens.long()[:, None, None]
    if bits is None:
        return inside & (n <= first + i[None, :, None])
    own_row = (n - first).clamp(0, 63)
    return inside & ((n < first) | (((bits[:, :, None] >> own_row) & 1) != 0))


def _plain_attention(s, prefix):
    q = s["q"]
    T, B = q.shape[0], s["lens"].shape[0]
    at, real = _padded(_row_ends(T, B, s["offsets"]), s["case"]["rows"])
    k, v = _rows_from_pages(s["k"], s["table"]), _rows_from_pages(s["v"], s["table"])
    i = torch.arange(at.shape[1], device="cuda")
    sees = _sees(s["lens"], real.sum(1), i, k.shape[2], None if s["bits"] is None else s["bits"][at])
    if prefix:
        g = torch.repeat_interleave(torch.arange(s["prefix_lens"].shape[0], device="cuda"),
                                    (s["groups"][1:] - s["groups"][:-1]).long(), output_size=B)
        kp = _rows_from_pages(s["k"], s["prefix_table"])
        vp = _rows_from_pages(s["v"], s["prefix_table"])
        k, v = torch.cat([kp[g], k], 2), torch.cat([vp[g], v], 2)
        there = torch.arange(kp.shape[2], device="cuda")[None] < s["prefix_lens"][g].long()[:, None]
        sees = torch.cat([there[:, None].expand(B, at.shape[1], -1), sees], 2)
    o = _attend(q[at], k, v, sees)
    out = torch.zeros((T + 1, *q.shape[1:]), dtype=q.dtype, device="cuda")
    out[torch.where(real, at, T)] = o.to(q.dtype)  # what pads goes to a row behind the last
    return out[:T]


def _plain_append(s):
    q, kn, vn = s["q"].float(), s["kn"].float(), s["vn"].float()
    T, D, page = q.shape[0], q.shape[2], s["k"].shape[2]
    B = s["lens"].shape[0]
    o = _row_ends(T, B, s["offsets"])
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(o, t, right=True) - 1
    slot = s["lens"].long()[b] - o[b + 1] + t
    # angles in 64 bits: positions are far, a 32-bit product would lose the angle's fraction
    f = torch.exp(torch.arange(0, D, 2, device="cuda", dtype=torch.float64) * (-math.log(BASE) / D))
    angle = s["positions"].double()[:, None] * f[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def normed(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w

    def turned(x):
        a, c = x[..., : D // 2], x[..., D // 2:]
        return torch.cat([a * cos - c * sin, c * cos + a * sin], -1)

    k2 = turned(normed(kn, s["k_norm"])).to(s["k"].dtype)
    p = s["table"].long()[b, slot // page]
    s["k"][p, :, slot % page] = k2
    s["v"][p, :, slot % page] = vn.to(s["v"].dtype)
    return turned(normed(q, s["q_norm"])).to(s["k"].dtype), s["k"], s["v"]


def _plain_compact(s):
    page = s["k"].shape[3]
    B, m = s["keep"].shape
    i = torch.arange(m, device="cuda")[None].expand(B, m)
    taken = i < s["n_keep"][:, None]  # what is not taken moves the first row onto itself
    b = torch.arange(B, device="cuda")[:, None].expand(B, m)
    src = (s["starts"][:, None] + torch.where(taken, s["keep"], 0)).long()
    dst = (s["starts"][:, None] + torch.where(taken, i, 0)).long()
    ps, pd = s["table"].long()[b, src // page], s["table"].long()[b, dst // page]
    for_k, for_v = s["k"][:, ps, :, src % page], s["v"][:, ps, :, src % page]
    s["k"][:, pd, :, dst % page] = for_k
    s["v"][:, pd, :, dst % page] = for_v
    return s["k"], s["v"], s["starts"] + s["n_keep"]


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from woodcock_b200 import ops

        if op == "append":
            q = ops.paged_append(s["q"], s["kn"], s["vn"], s["k"], s["v"], s["table"], s["lens"],
                                 positions=s["positions"], q_offsets=s["offsets"], base=BASE, q_norm=s["q_norm"],
                                 k_norm=s["k_norm"], eps=EPS)
            return q, s["k"], s["v"]
        if op == "attention":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], q_offsets=s["offsets"],
                                       tree_mask=s["bits"])
        if op == "prefix":
            return ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix_lens"],
                                               s["groups"], s["table"], s["lens"], q_offsets=s["offsets"],
                                               tree_mask=s["bits"])
        lens = ops.paged_compact(s["k"], s["v"], s["table"], s["starts"], s["keep"], s["n_keep"])
        return s["k"], s["v"], lens
    if op == "append":
        return _plain_append(s)
    if op == "compact":
        return _plain_compact(s)
    return _plain_attention(s, op == "prefix")


# ---------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, page = case["op"], case["page"]
    if op == "compact":
        k, v = s["k"].double(), s["v"].double()
        for b in range(case["requests"]):
            start, row = int(s["starts"][b]), s["table"][b].tolist()
            for i, j in enumerate(s["keep"][b].tolist()):
                (ps, os), (pd, od) = divmod(start + j, page), divmod(start + i, page)
                k[:, row[pd], :, od] = k[:, row[ps], :, os].clone()
                v[:, row[pd], :, od] = v[:, row[ps], :, os].clone()
        return k, v, None
    rows, lens = _rows_of(case), _lens_of(case)
    q = s["q"].double()
    T, H, D = q.shape
    Hk = case["kv_heads"]
    table = s["table"].long()
    if op == "append":
        k, v = s["k"].double(), s["v"].double()
        f = BASE ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) * 2 / D)
        turn = torch.polar(torch.ones((T, D // 2), device="cuda", dtype=torch.float64),
                           s["positions"].double()[:, None] * f)[:, None]

        def rotated(x, w):
            x = x.double()
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            z = torch.complex(x[..., : D // 2], x[..., D // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        kr, vr = rotated(s["kn"], s["k_norm"]), s["vn"].double()
        t = 0
        for b, (r, n) in enumerate(zip(rows, lens)):
            slot = torch.arange(n - r, n, device="cuda")
            k[table[b, slot // page], :, slot % page] = kr[t: t + r]
            v[table[b, slot // page], :, slot % page] = vr[t: t + r]
            t += r
        return rotated(s["q"], s["q_norm"]), k, v

    def keys(pool, row, n):
        at = torch.arange(n, device="cuda")
        return pool[row[at // page], :, at % page].double().transpose(0, 1)  # [Hk][n][D]

    out = torch.zeros((T, H, D), device="cuda", dtype=torch.float64)
    t = 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        if n + case.get("prefix", 0):
            k, v = keys(s["k"], table[b], n), keys(s["v"], table[b], n)
            pre = 0
            if op == "prefix":
                row = s["prefix_table"][b // case["requests"]].long()
                pre = case["prefix"]
                k = torch.cat([keys(s["k"], row, pre), k], 1)
                v = torch.cat([keys(s["v"], row, pre), v], 1)
            for r0 in range(0, r, 512):
                r1 = min(r, r0 + 512)
                i = torch.arange(r0, r1, device="cuda")[:, None]
                j = torch.arange(-pre, n, device="cuda")[None] - (n - r)  # key's number among the new rows
                if case["mask"] == "tree":
                    hidden = (j >= 0) & (((s["bits"][t + r0: t + r1, None] >> j.clamp(min=0)) & 1) == 0)
                else:
                    hidden = j > i
                for h in range(H):
                    z = q[t + r0: t + r1, h] @ k[h // (H // Hk)].T / math.sqrt(D)
                    w = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                    out[t + r0: t + r1, h] = w @ v[h // (H // Hk)]
        t += r
    return out
