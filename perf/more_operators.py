"""Operators of long sessions and beam searches over the paged cache, case by case: the attention weight
that each key gathers, eviction by it, beam selection, reordering of the beams' pages.

A long session keeps a key's share of the attention (summed over the rows and query heads that look at
it) beside the key, in pages of its own; when a request outgrows its budget the keys with the largest
sums stay, with the first and the last ones. A beam search picks the best continuations over beams and
vocabulary and hands every new beam its parent's history: full pages are shared by page number, the page
that is still being filled is copied for every further child of a parent.

``run`` computes a case in elementary torch operations, or (``own``) through ``woodcock_b200.ops``.

Layout: pages [layers][pages][kv_heads][page_size][head_dim], mass pages the same without head_dim, fp32.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------- the cases


def listed():
    tall = {"heads": 16, "kv_heads": 8, "head_dim": 128}   # the 1.7B layout
    wide = {"heads": 32, "kv_heads": 8, "head_dim": 128}   # the 4B layout
    tiny = {"heads": 4, "kv_heads": 2, "head_dim": 64}     # the tiny fp32 model
    pages = {"kv_heads": 8, "head_dim": 128, "dtype": "bf16"}
    return [
        # one session, one token: the latency of a step
        {"name": "mass decode 1", "op": "mass", **tall, "dtype": "bf16", "requests": 1, "rows": 1, "ragged": False,
         "len": 513, "page": 16, "add": True},
        # 64 sessions of very unequal length, one token each, an idle slot among them
        {"name": "mass decode 64 ragged", "op": "mass", **wide, "dtype": "bf16", "requests": 64, "rows": 1,
         "ragged": True, "len": 12289, "page": 16, "add": True},
        # the accepted rows of eight chains, fp32
        {"name": "mass chains fp32", "op": "mass", **tiny, "dtype": "fp32", "requests": 8, "rows": 5, "ragged": False,
         "len": 600, "page": 16, "add": True},
        # the last rows of long prompts judge the keys before them: the window that looks back
        {"name": "mass window 8x32", "op": "mass", **wide, "dtype": "bf16", "requests": 8, "rows": 32, "ragged": False,
         "len": 16384, "page": 64, "add": False},
        # all rows of prompts of unequal length
        {"name": "mass prompts ragged", "op": "mass", **wide, "dtype": "bf16", "requests": 4, "rows": 4096,
         "ragged": True, "len": 4096, "page": 64, "add": True},
        # one session outgrows its budget, every layer
        {"name": "evict 1", "op": "evict", **pages, "layers": 28, "requests": 1, "len": 640, "ragged": False,
         "budget": 512, "sinks": 4, "recent": 64, "page": 16},
        # a batch after its prompts: some within the budget, some far over it
        {"name": "evict 32 ragged", "op": "evict", **pages, "layers": 4, "requests": 32, "len": 8191, "ragged": True,
         "budget": 2048, "sinks": 4, "recent": 128, "page": 64},
        # one search of four beams over the full vocabulary, twice as many candidates as beams
        {"name": "select 1x4", "op": "select", "requests": 1, "beams": 4, "vocab": 151936, "n": 8, "dtype": "fp32",
         "state": "running"},
        # a batch of searches
        {"name": "select 64x8", "op": "select", "requests": 64, "beams": 8, "vocab": 151936, "n": 16, "dtype": "fp32",
         "state": "running"},
        # wide beams over a trimmed head whose logits stay bf16, a part of the beams at their end
        {"name": "select 16x32 trimmed", "op": "select", "requests": 16, "beams": 32, "vocab": 16384, "n": 64,
         "dtype": "bf16", "state": "finished"},
        # one search of four beams, two of them die, every layer
        {"name": "reorder 1x4", "op": "reorder", **pages, "layers": 28, "requests": 1, "beams": 4, "live": 2,
         "prompt": 640, "len": 650, "page": 16},
        # a batch of searches, three beams of eight die in each, every layer
        {"name": "reorder 32x8", "op": "reorder", **pages, "layers": 28, "requests": 32, "beams": 8, "live": 5,
         "prompt": 384, "len": 509, "page": 64},
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
    return {k: v for k, v in listed()[0].items() if k != "name"} | {"len": rng.randrange(2, 4000)}


def _drawn(rng, s):
    def upto(lo, hi):
        return _log_int(rng, lo, max(lo, int(hi * s)))

    op = rng.choice(["mass", "mass", "evict", "select", "select", "reorder"])
    if op == "select":
        c = {"op": op, "beams": upto(1, 32), "vocab": upto(50, 152064), "dtype": rng.choice(["fp32", "fp32", "bf16"]),
             "state": rng.choice(["running", "running", "first", "finished"])}
        c["requests"] = upto(1, max(1, 60_000_000 // (c["beams"] * c["vocab"])) if c["vocab"] > 4000 else 64)
        c["requests"] = min(c["requests"], 128)
        c["n"] = min(64, rng.choice([c["beams"], 2 * c["beams"], rng.randrange(1, 65)]))
        return c
    heads, kv = rng.choice([(16, 8), (32, 8), (4, 2), (8, 8), (8, 1), (40, 8), (6, 2)])
    c = {"op": op, "heads": heads, "kv_heads": kv, "head_dim": rng.choice([64, 128, 128]),
         "dtype": rng.choice(["bf16", "bf16", "bf16", "fp32"]), "page": rng.choice([16, 32, 64, 128])}
    small = c["dtype"] == "fp32"
    if op == "mass":
        kind = rng.choice(["decode", "chain", "window", "prompt"])
        c |= {"ragged": rng.random() < 0.5, "add": rng.random() < 0.7}
        if kind == "decode":
            c |= {"requests": upto(1, 96), "rows": 1}
            c["len"] = upto(1, (40000 if small else 300000) // c["requests"])
        elif kind == "chain":
            c |= {"requests": upto(1, 64), "rows": rng.randrange(2, 10)}
            c["len"] = c["rows"] + upto(1, (20000 if small else 200000) // c["requests"])
        elif kind == "window":
            c |= {"requests": upto(1, 16), "rows": rng.randrange(10, 65)}
            c["len"] = c["rows"] + upto(1, (10000 if small else 100000) // c["requests"])
        else:
            c |= {"requests": upto(1, 4), "rows": upto(65, 600 if small else 3000)}
            c["len"] = c["rows"] + rng.choice([0, 0, rng.randrange(0, 2000)])
        return c
    del c["heads"]
    if op == "evict":
        c |= {"layers": upto(1, 36), "requests": upto(1, 48), "ragged": rng.random() < 0.6, "sinks": rng.choice([0, 1, 4, 17])}
        c["len"] = upto(2, max(2, min(40000, (400_000 if small else 800_000) // (c["layers"] * c["requests"]))))
        c["budget"] = max(1, int(c["len"] * rng.uniform(0.1, 1.0)))
        c["sinks"] = min(c["sinks"], c["budget"])
        c["recent"] = rng.randrange(0, c["budget"] - c["sinks"] + 1) if rng.random() < 0.8 else 0
    else:
        c |= {"layers": upto(1, 36), "requests": upto(1, 32), "beams": upto(1, 16)}
        c["live"] = rng.randrange(1, c["beams"] + 1)
        c["prompt"] = rng.randrange(0, 800)
        c["len"] = c["prompt"] + rng.randrange(0, 200)
    return c


# ---------------------------------------------------------------------------- sizes


def _rows_of(case):
    """New rows of each request: all alike, or from one up to ``rows``."""
    B, n = case["requests"], case["rows"]
    if not case["ragged"] or n == 1:
        return [n] * B
    return [max(1, n if i == 0 else int(n * ((i * 0.6180339887) % 1.0))) for i in range(B)]


def _lens_of(case):
    """Keys of each request, its new rows included. Ragged: spread from short to ``len``; from three
    requests on, the last of a one-row batch is an idle slot (no keys)."""
    B, n = case["requests"], case["len"]
    least = _rows_of(case) if case["op"] == "mass" else [1] * B
    if not case["ragged"]:
        return [max(n, r) for r in least]
    lens = [max(r, n if i == 0 else int(n * ((i * 0.7548776662) % 1.0))) for i, r in enumerate(least)]
    if case["op"] == "mass" and case["rows"] == 1 and B >= 3:
        lens[-1] = 0
    return lens


def _budgets_of(case):
    """Ragged: the requests' budgets differ by up to a fifth, none below what is protected."""
    B, n = case["requests"], case["budget"]
    if not case["ragged"]:
        return [n] * B
    return [max(case["sinks"] + case["recent"], 1, n - i * 7 % max(1, n // 5)) for i in range(B)]


def _search_lens(case):
    """Keys of each request's beams: around ``len``, the prompt at least."""
    return [max(case["prompt"], 1, case["len"] - i * 5 % 41) for i in range(case["requests"])]


def work(case):
    if case["op"] == "select":
        e = 2 if case["dtype"] == "bf16" else 4
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * e + 4) + case["requests"] * case["n"] * 12, "flops": 3 * rows * case["vocab"]}
    D, Hk = case["head_dim"], case["kv_heads"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "mass":
        # K and the rows once; sums are read (where they are added to) and written
        H, T = case["heads"], sum(_rows_of(case))
        keys, seen = 0, 0
        for r, n in zip(_rows_of(case), _lens_of(case)):
            keys += n
            seen += r * (n - r) + r * (r + 1) // 2 if n else 0
        return {"bytes": keys * Hk * (D * e + (8 if case["add"] else 4)) + T * H * D * e, "flops": 2 * seen * H * D}
    if case["op"] == "evict":
        # the sums once; what is behind the first rows is read and written, K, V and its sum
        total = 0
        for n, m in zip(_lens_of(case), _budgets_of(case)):
            if n > m:
                total += n * 4 + (m - case["sinks"]) * 2 * (2 * D * e + 4)
        return {"bytes": max(total * case["layers"] * Hk, 8 * case["requests"]), "flops": 0}
    # reorder: the partial page of a parent with further children is read once and written for each of them
    extra = case["beams"] - case["live"]
    rows = sum(n % case["page"] for n in _search_lens(case))
    cols = max(-(-n // case["page"]) for n in _search_lens(case))
    moved = rows * case["layers"] * Hk * 2 * D * e
    return {"bytes": moved * (extra + min(extra, case["live"])) + 8 * case["requests"] * case["beams"] * (cols + 1), "flops": 0}


def _cost(case):
    w = work(case)
    # fp32 products run without the matrix units
    return max(w["bytes"] / 6.4e12, w["flops"] / (1.6e15 if case.get("dtype") == "bf16" else 4e13))


# ---------------------------------------------------------------------------- inputs


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return _ints(out)


def _table(gen, lens, page):
    """A page table whose pages are scattered over the pool, and the number of pages."""
    width = max(1, max(-(-n // page) for n in lens))
    order = torch.randperm(len(lens) * width, generator=gen, device="cuda")
    return order.reshape(len(lens), width).to(torch.int32), len(lens) * width


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    def pool(*shape):
        return torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)

    s = {"case": dict(case)}
    B = case["requests"]
    if case["op"] == "select":
        W, V = case["beams"], case["vocab"]
        # a head's logits: wide noise, and a few tokens that stand out
        z = randn(B, W, V, scale=2.5)
        few = torch.randint(0, V, (B, W, 8), generator=gen, device="cuda")
        z.scatter_add_(2, few, 6 + randn(B, W, 8, scale=2.0))
        s["logits"] = z.to(DTYPES[case["dtype"]])
        scores = -(8 + 6 * torch.rand((B, W), generator=gen, device="cuda")).sort(1).values
        if case["state"] == "first":
            scores[:, 0] = 0.0
            scores[:, 1:] = -math.inf
        s["scores"] = scores
        s["finished"] = torch.rand((B, W), generator=gen, device="cuda") < 0.25 if case["state"] == "finished" else None
        s["pad"] = V // 2
        return s
    Hk, D, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "mass":
        H, rows, lens = case["heads"], _rows_of(case), _lens_of(case)
        s["lens"] = _ints(lens)
        s["offsets"] = _offsets(rows) if case["ragged"] else None
        s["table"], pages = _table(gen, lens, page)
        # normalised keys, queries somewhat longer, so that some keys stand out
        s["q"] = randn(sum(rows), H, D, dtype=DTYPES[case["dtype"]], scale=1.5)
        s["k"] = pool(pages, Hk, page, D)
        s["mass"] = randn(pages, Hk, page).exp_()
        return s
    L = case["layers"]
    if case["op"] == "evict":
        lens = _lens_of(case)
        s["lens"] = _ints(lens)
        s["table"], pages = _table(gen, lens, page)
        s["budget"] = _ints(_budgets_of(case)) if case["ragged"] else case["budget"]
        s["k"], s["v"] = pool(L, pages, Hk, page, D), pool(L, pages, Hk, page, D)
        # a few keys gather most of the weight
        s["mass"] = randn(L, pages, Hk, page, scale=2.0).exp_()
        return s
    # reorder: the beams of a request share the prompt's full pages and have pages of their own behind them
    W, lens = case["beams"], _search_lens(case)
    shared = case["prompt"] // page
    width = max(1, max(n // page + 1 for n in lens))
    tail = width - shared
    order = torch.randperm(B * (shared + W * tail), generator=gen, device="cuda").to(torch.int32)
    common = order[: B * shared].view(B, 1, shared).expand(B, W, shared)
    s["table"] = torch.cat([common, order[B * shared:].view(B, W, tail)], 2).reshape(B * W, width).contiguous()
    s["lens"] = _ints([n for n in lens for _ in range(W)])
    # the survivors, and their further children one for each in turn, in any order
    alive = torch.rand((B, W), generator=gen, device="cuda").argsort(1)[:, : case["live"]]
    child = alive[:, torch.arange(W, device="cuda") % case["live"]]
    s["parents"] = child.gather(1, torch.rand((B, W), generator=gen, device="cuda").argsort(1)).to(torch.int32)
    s["k"], s["v"] = pool(L, order.numel(), Hk, page, D), pool(L, order.numel(), Hk, page, D)
    return s


# ---------------------------------------------------------------------------- the plain forms


def _plain_mass(s):
    q, table, lens, page = s["q"], s["table"].long(), s["lens"].long(), s["k"].shape[2]
    T, H, D = q.shape
    B, Hk = table.shape[0], s["k"].shape[1]
    rep = H // Hk
    o = torch.arange(0, T + 1, T // B, device="cuda") if s["offsets"] is None else s["offsets"].long()
    n = o[1:] - o[:-1]
    i = torch.arange(s["case"]["rows"], device="cuda")
    real = i[None] < n[:, None]
    at = torch.where(real, o[:-1, None] + i[None], 0)
    k = s["k"][table].permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D).float()  # [B][Hk][N][D]
    N, R = k.shape[2], at.shape[1]
    j = torch.arange(N, device="cuda")
    sees = real[:, :, None] & (j <= (lens - n)[:, None, None] + i[None, :, None]) & (j < lens[:, None, None])
    qh = q[at].float().view(B, R, Hk, rep, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, rep * R, D)
    z = (qh @ k.transpose(2, 3)).view(B, Hk, rep, R, N).mul_(D ** -0.5)
    z.masked_fill_(~sees[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    z.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    z.div_(z.sum(-1, keepdim=True).clamp_(min=1e-30))
    more = z.sum((2, 3)).transpose(1, 2)  # [B][N][Hk]
    # a key that is new in this call starts from nothing
    p, r = table[:, j // page], (j % page).expand(B, N)
    was = s["mass"][p, :, r]
    new = (j >= (lens - n)[:, None])[..., None] if s["case"]["add"] else torch.ones((1, 1, 1), dtype=torch.bool, device="cuda")
    s["mass"][p, :, r] = torch.where((j < lens[:, None])[..., None], torch.where(new, 0.0, was) + more, was)
    return s["mass"]


def _plain_evict(s):
    c, page = s["case"], s["k"].shape[3]
    table, lens = s["table"].long(), s["lens"].long()
    B, L, Hk = table.shape[0], s["k"].shape[0], s["k"].shape[2]
    m = torch.as_tensor(s["budget"], device="cuda").long().expand(B)
    over = lens > m
    w = s["mass"][:, table].transpose(2, 3).reshape(L, B, Hk, -1).clone()  # [L][B][cols][Hk][page] -> [L][B][Hk][N]
    N = w.shape[3]
    j = torch.arange(N, device="cuda")
    w.masked_fill_(((j < c["sinks"]) | (j >= (lens - c["recent"])[:, None]))[None, :, None], math.inf)
    w.masked_fill_((j >= lens[:, None])[None, :, None], -math.inf)
    M = min(N, int(max(_budgets_of(c))))
    i = torch.arange(M, device="cuda")
    taken = over[:, None] & (i < m[:, None])
    order = w.sort(dim=-1, descending=True, stable=True).indices[..., :M]
    src = torch.where(taken[None, :, None], order, N).sort(-1).values
    # what is not taken repeats the first move, or moves the first row onto itself
    src = torch.where(taken[None, :, None], src, torch.where(over[None, :, None, None], src[..., :1], 0))
    dst = torch.where(taken, i, 0)
    b = torch.arange(B, device="cuda")[None, :, None, None]
    ell, h = torch.arange(L, device="cuda")[:, None, None, None], torch.arange(Hk, device="cuda")[None, None, :, None]
    ps, pd = table[b, src // page], table[b, (dst // page)[None, :, None]]
    rs, rd = src % page, (dst % page)[None, :, None]
    for x in (s["k"], s["v"], s["mass"]):
        x[ell, pd, h, rd] = x[ell, ps, h, rs]
    return s["k"], s["v"], s["mass"], torch.minimum(lens, m).to(torch.int32)


def _plain_select(s):
    z = s["logits"]
    B, W, V = z.shape
    n, c = s["case"]["n"], min(s["case"]["n"], V)
    z = z.float() + 0.0
    # in 64 bits: neighbours in rank may lie closer than a 32-bit sum tells apart
    d = z.double()
    top = d.amax(-1, keepdim=True)
    lse = (d - top).exp_().sum(-1, keepdim=True).log_() + top
    del d
    # each beam's best, ties to the lowest token: the logits' order as integers, the token below it
    bits = z.view(torch.int32).long()
    bits = torch.where(bits < 0, -0x80000000 - bits, bits)
    best = (bits * V + (V - 1 - torch.arange(V, device="cuda"))).topk(c, -1).values
    token = V - 1 - best % V
    score = s["scores"].double()[:, :, None] + (z.gather(-1, token).double() - lse)
    if s["finished"] is not None:  # a beam at its end is carried on as it is
        f = s["finished"][:, :, None]
        first = torch.arange(c, device="cuda") == 0
        score = torch.where(f, torch.where(first, s["scores"].double()[:, :, None], -math.inf), score)
        token = torch.where(f, s["pad"], token)
    parent = torch.arange(W, device="cuda")[None, :, None].expand(B, W, c)
    # ties between beams: the lower beam first (a beam's own are in the tokens' order)
    score, at = score.reshape(B, -1).sort(dim=-1, descending=True, stable=True)
    parent, token = parent.reshape(B, -1).gather(1, at), token.reshape(B, -1).gather(1, at)
    none = score == -math.inf
    out = [torch.where(none, x, y) for x, y in ((-math.inf, score), (0, parent), (0, token))]
    if out[0].shape[1] < n:
        more = n - out[0].shape[1]
        out = [torch.nn.functional.pad(x, (0, more), value=v) for x, v in zip(out, (-math.inf, 0, 0))]
    return out[0][:, :n].float(), out[1][:, :n].to(torch.int32), out[2][:, :n].to(torch.int32)


def _plain_reorder(s):
    page, B = s["k"].shape[3], s["case"]["requests"]
    W = s["case"]["beams"]
    table = s["table"].view(B, W, -1)
    cols = table.shape[2]
    parents, lens = s["parents"].long(), s["lens"].view(B, W)[:, 0].long()
    w = torch.arange(W, device="cuda")
    same = parents[:, :, None] == parents[:, None]
    further = (same & (w[None] < w[:, None])).any(2)  # an earlier beam has the same parent
    dead = ~(parents[:, :, None] == w).any(1)
    # the i-th further child takes the i-th dead beam's page
    graves = torch.where(dead, w, W).sort(1).values
    grave = graves.gather(1, (further.cumsum(1) - 1).clamp_(min=0)).clamp_(max=W - 1)
    col = torch.arange(cols, device="cuda")[None, None]
    full, part = (lens // page)[:, None, None], ((lens % page) > 0)[:, None, None]
    heir = torch.where(further, grave, parents)
    old = table.gather(1, parents[:, :, None].expand(B, W, cols))
    filled = table.gather(1, heir[:, :, None].expand(B, W, cols))
    new = torch.where(col < full, old, torch.where((col == full) & part, filled, table))
    # rows of the page being filled, for every further child
    at = full[:, :, 0].clamp(max=cols - 1).expand(B, W)[:, :, None]
    ps, pd = old.gather(2, at)[..., 0].long(), filled.gather(2, at)[..., 0].long()
    r = torch.arange(page, device="cuda")
    rows = r[None, None] < (lens % page)[:, None, None]
    keep = (further[:, :, None] & rows).reshape(-1).nonzero()[:, 0]
    ps, pd = (x[:, :, None].expand(B, W, page).reshape(-1)[keep] for x in (ps, pd))
    rr = r.expand(B, W, page).reshape(-1)[keep]
    for x in (s["k"], s["v"]):
        x[:, pd, :, rr] = x[:, ps, :, rr]
    return s["k"], s["v"], new.reshape(B * W, cols).contiguous()


def run(state):
    s = state
    c = s["case"]
    if own:
        from woodcock_b200 import ops

        if c["op"] == "mass":
            return ops.paged_mass(s["q"], s["k"], s["mass"], s["table"], s["lens"], q_offsets=s["offsets"], add=c["add"])
        if c["op"] == "evict":
            lens = ops.paged_evict(s["k"], s["v"], s["mass"], s["table"], s["lens"], s["budget"], sinks=c["sinks"],
                                   recent=c["recent"])
            return s["k"], s["v"], s["mass"], lens
        if c["op"] == "select":
            return ops.beam_select(s["logits"], s["scores"], c["n"], finished=s["finished"], pad=s["pad"])
        table = ops.beam_reorder(s["k"], s["v"], s["table"], s["lens"], s["parents"])
        return s["k"], s["v"], table
    return {"mass": _plain_mass, "evict": _plain_evict, "select": _plain_select, "reorder": _plain_reorder}[c["op"]](s)


# ---------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "select":
        B, W, n = case["requests"], case["beams"], case["n"]
        best = torch.full((B, n), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            row = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
            if s["finished"] is not None:
                for w in s["finished"][b].nonzero()[:, 0].tolist():
                    row[w] = -math.inf
                    row[w, s["pad"]] = s["scores"][b, w].double()
            t = row.flatten().topk(min(n, row.numel())).values
            best[b, : t.numel()] = t
        return best, None, None
    page, table = case["page"], s["table"].long()
    if op == "mass":
        rows, lens = _rows_of(case), _lens_of(case)
        H, Hk = case["heads"], case["kv_heads"]
        mass, q = s["mass"].double(), s["q"].double()
        t = 0
        for b, (r, n) in enumerate(zip(rows, lens)):
            slot = torch.arange(n, device="cuda")
            where = (table[b, slot // page], slice(None), slot % page)
            k = s["k"][where].double()  # [n][Hk][D]
            got = mass[where]
            got[n - r if case["add"] else 0:] = 0
            for r0 in range(0, r if n else 0, 512):
                r1 = min(r, r0 + 512)
                hidden = slot[None] > torch.arange(n - r + r0, n - r + r1, device="cuda")[:, None]
                for h in range(H):
                    z = q[t + r0: t + r1, h] @ k[:, h // (H // Hk)].T / math.sqrt(case["head_dim"])
                    got[:, h // (H // Hk)] += torch.softmax(z.masked_fill(hidden, -math.inf), -1).sum(0)
            mass[where] = got
            t += r
        return mass
    k, v = s["k"].double(), s["v"].double()
    if op == "evict":
        mass = s["mass"].double()
        for b, (n, m) in enumerate(zip(_lens_of(case), _budgets_of(case))):
            if n <= m:
                continue
            lo, hi = case["sinks"], n - case["recent"]
            slot = torch.arange(n, device="cuda")
            for layer in range(case["layers"]):
                for h in range(case["kv_heads"]):
                    here = (layer, table[b, slot // page], h, slot % page)
                    rank = mass[here][lo:hi].argsort(descending=True, stable=True)[: m - lo - case["recent"]]
                    kept = torch.cat([slot[:lo], lo + rank.sort().values, slot[hi:]])
                    for x in (k, v, mass):
                        got = x[here]
                        got[:m] = got[kept]
                        x[here] = got
        return k, v, mass, None
    W = case["beams"]
    for b, n in enumerate(_search_lens(case)):
        parents, rest, col = s["parents"][b].tolist(), n % page, n // page
        free, taken = [w for w in range(W) if w not in parents], set()
        for p in parents:
            if p in taken and rest:
                src, dst = int(table[b * W + p, col]), int(table[b * W + free.pop(0), col])
                k[:, dst, :, :rest] = k[:, src, :, :rest]
                v[:, dst, :, :rest] = v[:, src, :, :rest]
            taken.add(p)
    return k, v, None
