"""The paged operators against a plain implementation in 64 bits.

Tolerances. One rounding to a type is off by at most h = finfo(type).eps / 2 of the value (bf16: 2^-8).
* Attention, bf16 pages: the weights are rounded once (h of each term's magnitude), the output once (h
  of the output), and the scores, statistics and sums are fp32: h |o| + (h + 2^-12) sum p |v|.
  2^-12 covers the fp32 terms: a score is a sum of head_dim products, off by at most
  (head_dim + 4) 2^-24 sum |q k| scale, and shifts its weight by as much (sum |q k| scale < 120 here:
  132 * 120 * 2^-24 < 2^-10 at the very worst, its usual size 2^-15; the worst is added as `es`).
* Attention, fp32 pages: the same terms without roundings to bf16: (2 es + n 2^-24 + 2^-19) sum p |v|,
  n keys; 2^-19 covers exp2f (2 ulp) on both sides, scale * log2(e) rounded once (|s| < 40) and l.
* Append: normalisation sums head_dim squares (head_dim 2^-24 relative at worst, half of it after the
  root), the rotation's cosine and sine are within 2^-21, products and the sum add 2^-22:
  (|a| + |b|) (head_dim 2^-25 + 2^-20), and h of the result where it is rounded to bf16.
* Compaction moves bits.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def half_step(dt):
    return torch.finfo(dt).eps / 2


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(rows):
    return i32([0, *torch.tensor(rows).cumsum(0).tolist()])


class Case:
    """A pool with scattered pages; everything that no key lies in holds NaN."""

    def __init__(self, seed, lens, rows, H, Hk, D, page, dtype, layout="heads", prefix=(), spare=1):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.rows, self.H, self.Hk, self.D, self.page, self.dtype = lens, rows, H, Hk, D, page, dtype
        self.prefix = list(prefix)
        need = [-(-n // page) for n in [*lens, *self.prefix]]
        width = max([1, *need[: len(lens)]])
        pwidth = max([1, *need[len(lens):]]) if self.prefix else 0
        total = len(lens) * width + len(self.prefix) * pwidth + spare
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        self.table = ids[: len(lens) * width].view(len(lens), width)
        self.ptable = ids[len(lens) * width: len(lens) * width + len(self.prefix) * pwidth].view(len(self.prefix), pwidth) \
            if self.prefix else None
        shape = (total, Hk, page, D) if layout == "heads" else (total, page, Hk, D)
        self.k = torch.full(shape, math.nan, dtype=dtype, device="cuda")
        self.v = torch.full(shape, math.nan, dtype=dtype, device="cuda")
        if layout != "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for t, ns in ((self.table, lens), (self.ptable, self.prefix)):
            for b, n in enumerate(ns):
                if n:
                    at = torch.arange(n, device="cuda")
                    p, r = t[b].long()[at // page], at % page
                    self.k[p, :, r] = self.randn(n, Hk, D)
                    self.v[p, :, r] = self.randn(n, Hk, D)
        self.q = self.randn(sum(rows), H, D, scale=1.5)
        self.off = offsets(rows)
        self.kv = i32(lens)

    def randn(self, *shape, scale=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * scale).to(self.dtype)

    def keys(self, pool, table, b, n):
        at = torch.arange(n, device="cuda")
        return pool[table[b].long()[at // self.page], :, at % self.page].double()  # [n][Hk][D]


def want_rows(c, b, t0, bits=None, group=None):
    """The formula in 64 bits for request b: output, sum p |v| and the score error's bound."""
    n, r = c.lens[b], c.rows[b]
    k, v = c.keys(c.k, c.table, b, n), c.keys(c.v, c.table, b, n)
    pre = 0
    if group is not None:
        pre = c.prefix[group]
        k = torch.cat([c.keys(c.k, c.ptable, group, pre), k])
        v = torch.cat([c.keys(c.v, c.ptable, group, pre), v])
    rep = c.H // c.Hk
    q = c.q[t0: t0 + r].double()
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    j = torch.arange(-pre, n, device="cuda")[None] - (n - r)
    i = torch.arange(r, device="cuda")[:, None]
    if bits is None:
        sees = j <= i
    else:
        sees = (j < 0) | ((bits[t0: t0 + r, None] >> j.clamp(0, 63)) & 1 != 0)
    # the prefix is seen whole, also by rows that have no slot of their own (fewer keys than new rows)
    sees = sees | (torch.arange(pre + n, device="cuda")[None] < pre)
    sees = sees[:, None].expand(r, c.H, -1)
    s = torch.einsum("rhd,khd->rhk", q, k) * c.D ** -0.5
    mag = torch.einsum("rhd,khd->rhk", q.abs(), k.abs()) * c.D ** -0.5
    s = torch.where(sees, s, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(sees, p, 0.0)  # rows that see nothing: 0
    v = torch.where(sees.any(1).any(0)[:, None, None], v, 0.0)  # keys that nobody sees may hold anything
    # a key that only some rows see may hold NaN for the others: sum over the seen ones alone
    if torch.isfinite(v).all():
        o = torch.einsum("rhk,khd->rhd", p, v)
        a = torch.einsum("rhk,khd->rhd", p, v.abs())
    else:
        o = torch.stack([torch.where(sees[x][..., None], p[x][..., None] * v.transpose(0, 1), 0.0).sum(1)
                         for x in range(r)])
        a = o.abs() + 1
    es = (c.D + 4) * 2.0 ** -24 * torch.where(sees, mag, 0.0).amax(-1, keepdim=True) if n + pre else \
        torch.zeros((r, c.H, 1), device="cuda", dtype=torch.float64)
    return o, a, es, n + pre


def check(c, out, bits=None, groups=None, only=None):
    h = half_step(c.dtype)
    t0 = 0
    for b, r in enumerate(c.rows):
        if r and (only is None or b == only):
            g = None if groups is None else next((g for g in range(len(groups) - 1) if groups[g] <= b < groups[g + 1]), None)
            o, a, es, n = want_rows(c, b, t0, bits, g)
            got = out[t0: t0 + r].double()
            if c.dtype is BF:
                tol = h * o.abs() + (h + 2.0 ** -12 + 2 * es) * a
            else:
                tol = (2 * es + n * 2.0 ** -24 + 2.0 ** -19) * a
            bad = (got - o).abs() > tol + 1e-30
            assert torch.isfinite(got).all() and not bad.any(), \
                f"request {b}: {int(bad.sum())} values off, worst {float(((got - o).abs() - tol).max()):.3g}"
        t0 += r


def tree_bits(rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for r in rows:
        anc = []
        for i in range(r):
            par = int(torch.randint(0, i, (1,), generator=g)) if i else -1
            anc.append((anc[par] if i else 0) | (1 << i))
        out += [x - (1 << 64) if x >> 63 else x for x in anc]
    return torch.tensor(out, dtype=torch.int64, device="cuda")


HEADS = [(16, 8, 128), (4, 2, 64), (8, 1, 128), (40, 8, 128), (3, 3, 64)]


# ------------------------------------------------------------------------------------------------ attention


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_lengths_around_tiles_and_pages(dtype, H, Hk, D, page):
    from woodcock_b200 import ops

    lens = [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 700, 1025]
    c = Case(1, lens, [1] * len(lens), H, Hk, D, page, dtype)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_long_request_is_divided_over_the_device(dtype):
    from woodcock_b200 import ops

    c = Case(2, [40001], [1], 16, 8, 128, 64, dtype)
    a = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    check(c, a)
    assert torch.equal(a, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))  # no order of arrival in the sums


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", HEADS)
def test_ragged_batch_of_steps_chains_and_prompts(dtype, H, Hk, D):
    from woodcock_b200 import ops

    rows = [1, 5, 130, 1, 0, 33, 300, 2]
    lens = [513, 200, 130, 1, 77, 290, 431, 900]
    c = Case(3, lens, rows, H, Hk, D, 32, dtype)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows, lens", [([700], [700]), ([257, 1023], [1500, 1023])])
def test_prompts(dtype, rows, lens):
    from woodcock_b200 import ops

    c = Case(4, lens, rows, 8, 2, 128, 64, dtype)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", HEADS)
@pytest.mark.parametrize("rows", [[16, 16, 16], [1, 64, 33], [5, 5]])
def test_tree_masks(dtype, H, Hk, D, rows):
    from woodcock_b200 import ops

    lens = [r + x for r, x in zip(rows, [0, 301, 77])]
    c = Case(5, lens, rows, H, Hk, D, 16, dtype)
    bits = tree_bits(rows)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off, tree_mask=bits), bits)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_see_nothing_give_zero(dtype):
    from woodcock_b200 import ops

    # no keys at all; more new rows than keys (the first see none); a tree row without bits or prefix
    c = Case(6, [0, 3, 40], [1, 5, 2], 16, 8, 128, 16, dtype)
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off)
    assert (out[0] == 0).all() and (out[1:3] == 0).all()
    check(c, out)
    c = Case(7, [4, 70], [4, 3], 8, 8, 64, 16, dtype)
    bits = tree_bits([4, 3])
    bits[2] = 0
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off, tree_mask=bits)
    assert (out[2] == 0).all()
    check(c, out, bits)
    # a table without a column: every request is empty
    empty = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    assert (ops.paged_attention(c.q[:2].contiguous(), c.k, c.v, empty, i32([0, 0])) == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [6, 48])
def test_masked_places_may_hold_anything(dtype, bad, rows):
    from woodcock_b200 import ops

    # tree: a node's K and V are poisoned; the rows that do not see it are as if it were not there
    c = Case(8, [rows + 90, rows], [rows, rows], 16, 8, 128, 16, dtype)
    bits = tree_bits(c.rows, 3)
    for b, n in enumerate(c.lens):
        node = n - rows + 3
        at = c.table[b].long()[node // 16], slice(None), node % 16
        c.k[at] = bad
        c.v[at] = bad
    blind = ((bits >> 3) & 1) == 0
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off, tree_mask=bits)
    for b, n in enumerate(c.lens):  # the reference with the node's place clean
        node = n - rows + 3
        at = c.table[b].long()[node // 16], slice(None), node % 16
        c.k[at] = 0
        c.v[at] = 0
    t0 = 0
    for b, r in enumerate(c.rows):
        o, a, es, n = want_rows(c, b, t0, bits)
        h = half_step(dtype)
        tol = (h * o.abs() + (h + 2.0 ** -12 + 2 * es) * a) if dtype is BF else (2 * es + n * 2.0 ** -24 + 2.0 ** -19) * a
        ok = blind[t0: t0 + r]
        assert ok.any()
        got = out[t0: t0 + r].double()
        assert ((got - o).abs() <= tol)[ok].all()
        t0 += r


@pytest.mark.parametrize("rows", [9, 200])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_later_row_of_a_prompt_does_not_reach_an_earlier_one(rows, dtype):
    from woodcock_b200 import ops

    c = Case(9, [rows + 20], [rows], 16, 8, 128, 16, dtype)
    key = 20 + rows // 2
    at = c.table[0].long()[key // 16], slice(None), key % 16
    clean = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    c.k[at] = math.nan
    c.v[at] = math.inf
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    assert torch.isfinite(out[: rows // 2]).all() and torch.isnan(out[rows // 2:].float()).all()
    tol = 2 * half_step(dtype) if dtype is BF else 2.0 ** -18
    assert (out[: rows // 2] - clean[: rows // 2]).abs().max() <= 4 * tol * clean.abs().max()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 40])
def test_strides_views_and_a_given_output(dtype, rows):
    from woodcock_b200 import ops

    c = Case(10, [100, rows, 333], [rows] * 3, 16, 8, 128, 32, dtype, layout="positions")
    T = 3 * rows
    fused = torch.full((T + 2, 32, 128), math.nan, dtype=dtype, device="cuda")
    fused[:T, 4:20] = c.q
    wide = torch.full((3, c.table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, : c.table.shape[1]] = c.table
    want = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    check(c, want)
    out = torch.full((T + 2, 16, 128), 5.0, dtype=dtype, device="cuda")
    # two rows behind the last request: neither read nor written
    got = ops.paged_attention(fused[:, 4:20], c.k, c.v, wide[:, : c.table.shape[1]], c.kv, q_offsets=c.off, out=out)
    assert got is out and torch.equal(got[:T], want) and (got[T:] == 5).all()
    odd = torch.empty(c.q.numel() + 1, dtype=dtype, device="cuda")[1:].view(c.q.shape)  # not 16-byte aligned
    odd.copy_(c.q)
    assert torch.equal(ops.paged_attention(odd, c.k, c.v, c.table, c.kv), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 40, 140])
def test_bad_pages_and_lengths_raise_the_error_word(dtype, rows):
    from woodcock_b200 import ops
    from woodcock_b200._lib import WC_ERR_DEVICE, WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    c = Case(11, [rows + 60, 300 + rows], [rows] * 2, 16, 8, 128, 16, dtype)
    want = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    ctx.synchronize()
    for entry in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = c.table.clone()
        t[0, 1] = entry
        out = ops.paged_attention(c.q, c.k, c.v, t, c.kv)
        torch.cuda.synchronize()
        with pytest.raises(WcError) as e:
            ctx.synchronize()
        assert e.value.status == WC_ERR_DEVICE
        assert torch.equal(out[rows:], want[rows:])  # the other request is not touched by it
    for n in (-5, c.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        out = ops.paged_attention(c.q, c.k, c.v, c.table, i32([n, c.lens[1]]))
        torch.cuda.synchronize()
        with pytest.raises(WcError):
            ctx.synchronize()
        # the lengths decide where the keys are cut, so the sums' order: held to the formula, not to the bits
        check(c, out, only=1)
    ctx.synchronize()


def test_offsets_that_are_no_offsets_stay_inside_the_buffers():
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    c = Case(12, [60, 90, 30], [4, 4, 4], 16, 8, 128, 16, BF)
    torch.cuda.synchronize()
    guard = torch.full((3, 12, 16, 128), 3.0, dtype=BF, device="cuda")
    for off in ([4, 0, 12, 8], [-9, 4, 8, 10 ** 9], [12, 8, 4, 0], [0, 0, 0, 0]):
        ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=i32(off), out=guard[1])
        ops.shared_prefix_attention(c.q, c.k, c.v, c.table, c.kv, i32([2, 0, 9, 1]), c.table, c.kv, q_offsets=i32(off),
                                    out=guard[1])
        torch.cuda.synchronize()
        assert (guard[0] == 3).all() and (guard[2] == 3).all()
    try:
        Context.get(0).synchronize()
    except RuntimeError:
        pass
    Context.get(0).synchronize()


def test_a_pool_whose_offsets_pass_32_bits():
    from woodcock_b200 import ops

    pages, page, Hk, D = 70_000, 64, 4, 128  # 2.3e9 elements a pool
    k = torch.empty((pages, Hk, page, D), dtype=BF, device="cuda")
    v = torch.empty_like(k)
    c = Case(13, [900], [1], 8, Hk, D, page, BF)
    far = torch.arange(pages - c.table.shape[1], pages, device="cuda")
    k[far], v[far] = c.k[c.table[0].long()], c.v[c.table[0].long()]
    got = ops.paged_attention(c.q, k, v, far.to(torch.int32)[None], c.kv)
    assert torch.equal(got, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))
    c2 = Case(13, [900], [140], 8, Hk, D, page, BF)
    k[far], v[far] = c2.k[c2.table[0].long()], c2.v[c2.table[0].long()]
    got = ops.paged_attention(c2.q, k, v, far.to(torch.int32)[None], c2.kv)
    assert torch.equal(got, ops.paged_attention(c2.q, c2.k, c2.v, c2.table, c2.kv))
    n = torch.randn((1, 4, D), device="cuda")
    ops.paged_append(torch.randn((1, 8, D), device="cuda"), n, n, k, v, far.to(torch.int32)[None], i32([900]))
    at = far[899 // page], slice(None), 899 % page
    assert torch.equal(v[at], n[0].to(BF))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", [(32, 1, 128), (71, 1, 64), (24, 2, 64)])
@pytest.mark.parametrize("rows", [1, 3, 37])
def test_many_query_heads_per_kv_head(dtype, H, Hk, D, rows):
    from woodcock_b200 import ops

    c = Case(50, [rows, 200, 97], [rows] * 3, H, Hk, D, 16, dtype)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))


@pytest.mark.parametrize("page", [16, 32, 128, 256])
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_of_every_size_on_the_tensor_cores(page, rows, D):
    from woodcock_b200 import ops

    c = Case(51, [rows, rows + 333, 2 * rows + 1], [rows] * 3, 16, 8, D, page, BF)
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 18])
def test_more_requests_than_a_block_has_threads(dtype, rows):
    from woodcock_b200 import ops

    B = 700
    lens = [(i * 37) % 90 + rows for i in range(B)]
    c = Case(52, lens, [rows] * B, 2, 1, 64, 16, dtype, prefix=[5 + i % 40 for i in range(350)])
    some = [0, 1, 255, 256, 383, 384, 511, 699]
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    for b in some:
        check_one(c, out, b, rows)
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off)
    for b in some:
        check_one(c, out, b, rows)
    groups = list(range(0, 701, 2))
    out = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32(c.prefix), i32(groups), c.table, c.kv, q_offsets=c.off)
    for b in some:
        check_one(c, out, b, rows, groups)


def check_one(c, out, b, rows, groups=None):
    """One request of a uniform batch, without the cost of all the others."""
    o, a, es, n = want_rows(c, b, b * rows, None, None if groups is None else b // 2)
    h = half_step(c.dtype)
    tol = (h * o.abs() + (h + 2.0 ** -12 + 2 * es) * a) if c.dtype is BF else (2 * es + n * 2.0 ** -24 + 2.0 ** -19) * a
    assert ((out[b * rows: (b + 1) * rows].double() - o).abs() <= tol + 1e-30).all(), b


@pytest.mark.parametrize("dtype", [BF, F32])
def test_trees_with_fewer_keys_than_rows_and_with_too_many_rows(dtype):
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    # rows without a slot: bit i still names new row i, whose key may lie before the first
    c = Case(53, [2, 30], [4, 30], 16, 8, 128, 16, dtype)
    bits = tree_bits([4, 30])
    check(c, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off, tree_mask=bits), bits)
    Context.get(0).synchronize()
    c = Case(54, [90], [65], 16, 8, 128, 16, dtype)
    ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, tree_mask=torch.ones(65, dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(WcError):
        Context.get(0).synchronize()
    Context.get(0).synchronize()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [2, 30, 200])
def test_a_query_row_of_nan_stays_alone(dtype, rows):
    from woodcock_b200 import ops

    c = Case(55, [rows + 70] * 3, [rows] * 3, 16, 8, 128, 32, dtype)
    want = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    c.q[rows + 1, 5] = math.nan
    got = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    assert torch.isnan(got[rows + 1, 5].float()).all()
    got[rows + 1, 5] = want[rows + 1, 5]
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [33, 150])
def test_poisoned_values_in_many_items_and_long_contexts(rows):
    """Every request holds a later row of NaN: all items of a block are summed again, divided ones too."""
    from woodcock_b200 import ops

    B = 40
    lens = [rows + (4000 if b == 0 else 60 + b) for b in range(B)]
    c = Case(56, lens, [rows] * B, 8, 8, 128, 64, BF, prefix=[300])
    clean = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    joined = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32([300]), i32([0, B]), c.table, c.kv)
    hole = rows // 3
    for b, n in enumerate(lens):
        key = n - rows + hole
        at = c.table[b].long()[key // 64], slice(None), key % 64
        c.k[at] = math.nan
        c.v[at] = math.nan
    for want, got in ((clean, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)),
                      (joined, ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32([300]), i32([0, B]), c.table, c.kv))):
        want, got = want.view(B, rows, 8, 128).float(), got.view(B, rows, 8, 128).float()
        assert torch.isnan(got[:, hole:]).all()
        # both within the tolerance of the formula: the rounded weights' (2^-8 of sum p |v|, at most max |v|) on
        # one side and the output's rounding on both
        assert (got[:, :hole] - want[:, :hole]).abs().max() <= 2.0 ** -8 * 5.5 + 2.0 ** -7 * want.abs().max()


# ------------------------------------------------------------------------------------------------ shared prefixes


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", HEADS)
@pytest.mark.parametrize("rows", [1, 7, 40])
def test_shared_prefixes(dtype, H, Hk, D, rows):
    from woodcock_b200 import ops

    # groups of unequal size, an empty prefix, one without requests, requests outside every group
    lens = [rows + x for x in (0, 100, 3, 64, 17, 0, 250)]
    groups = [1, 3, 3, 6]
    c = Case(14, lens, [rows] * 7, H, Hk, D, 32, dtype, prefix=[333, 64, 0])
    for r in (None, c.off):
        out = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32(c.prefix), i32(groups), c.table, c.kv, q_offsets=r)
        check(c, out, groups=groups)
    bits = tree_bits(c.rows, 5)
    out = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32(c.prefix), i32(groups), c.table, c.kv, tree_mask=bits)
    check(c, out, bits, groups)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_shared_prefix_of_a_ragged_batch_and_prompts(dtype):
    from woodcock_b200 import ops

    rows, groups = [150, 1, 0, 33, 2], [0, 2, 5]
    c = Case(15, [150, 900, 5, 40, 2], rows, 16, 8, 128, 16, dtype, prefix=[1000, 129])
    out = torch.full((sum(rows) + 3, 16, 128), 5.0, dtype=dtype, device="cuda")
    q = torch.cat([c.q, c.q[:3]])
    got = ops.shared_prefix_attention(q, c.k, c.v, c.ptable, i32(c.prefix), i32(groups), c.table, c.kv,
                                      q_offsets=c.off, out=out)
    check(c, got, groups=groups)
    assert (out[sum(rows):] == 5).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prefix_alone_and_nothing_at_all(dtype):
    from woodcock_b200 import ops

    # no own keys: the first row's place has no slot, but it sees the prefix; and one that sees nothing
    c = Case(16, [0, 0], [1, 1], 16, 8, 128, 16, dtype, prefix=[50, 0])
    out = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32(c.prefix), i32([0, 1, 2]), c.table, c.kv)
    check(c, out, groups=[0, 1, 2])
    assert (out[1] == 0).all()
    none = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    c = Case(17, [40, 7], [1, 1], 16, 8, 128, 16, dtype)
    assert torch.equal(ops.shared_prefix_attention(c.q, c.k, c.v, none, i32([]), i32([0]), c.table, c.kv),
                       ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))


# ------------------------------------------------------------------------------------------------ append


def want_rotated(x, w, pos, base, eps):
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    f = base ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) * 2 / D)
    ang = pos.double()[:, None, None] * f
    a, b = x[..., : D // 2], x[..., D // 2:]
    y = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    m = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, m * (D * 2.0 ** -25 + 2.0 ** -20)


@pytest.mark.parametrize("src", [BF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H, Hk, D", HEADS)
@pytest.mark.parametrize("gains", [True, False])
def test_append(src, dtype, H, Hk, D, gains):
    from woodcock_b200 import ops

    rows, lens, page = [1, 0, 40, 3, 17], [130, 9, 40, 20, 64], 16
    c = Case(20, lens, rows, H, Hk, D, page, dtype)
    T = sum(rows)
    fused = torch.randn((T, (H + 2 * Hk) * D), generator=c.g, device="cuda").to(src)
    q, k, v = (fused[:, a * D: b * D].view(T, b - a, D) for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    qn, kn = (1 + 0.2 * torch.randn(D, device="cuda") if gains else None for _ in range(2))
    slots = torch.cat([torch.arange(n - r, n, device="cuda") for n, r in zip(lens, rows)])
    far = torch.arange(T, device="cuda", dtype=torch.int32) * 97_003  # up to six million
    for pos in (None, far):
        k0, v0 = c.k.clone(), c.v.clone()
        got = ops.paged_append(q, k, v, c.k, c.v, c.table, c.kv, positions=pos, q_offsets=c.off, base=1e6, q_norm=qn,
                               k_norm=kn, eps=1e-6)
        at = slots if pos is None else pos
        y, tol = want_rotated(q, qn, at, 1e6, 1e-6)
        h = half_step(BF) if dtype is BF else 0.0
        assert ((got.double() - y).abs() <= tol + h * y.abs()).all()
        y, tol = want_rotated(k, kn, at, 1e6, 1e-6)
        b = torch.repeat_interleave(torch.arange(5, device="cuda"), i32(rows).long())
        p = c.table.long()[b, slots // page]
        assert ((c.k[p, :, slots % page].double() - y).abs() <= tol + h * y.abs()).all()
        assert torch.equal(c.v[p, :, slots % page], v.to(dtype))
        k0[p, :, slots % page], v0[p, :, slots % page] = c.k[p, :, slots % page], c.v[p, :, slots % page]
        assert torch.equal(c.k.nan_to_num(7.0), k0.nan_to_num(7.0))  # nothing else was written
        assert torch.equal(c.v.nan_to_num(7.0), v0.nan_to_num(7.0))


def test_append_agrees_with_the_contiguous_operators():
    from woodcock_b200 import ops

    c = Case(21, [50, 7], [3, 3], 16, 8, 128, 16, F32)
    q, k, v = c.q, c.randn(6, 8, 128), c.randn(6, 8, 128)
    w = 1 + 0.1 * torch.randn(128, device="cuda")
    pos = i32([47, 48, 49, 4, 5, 6])
    got = ops.paged_append(q, k, v, c.k, c.v, c.table, c.kv, base=1e6, q_norm=w, k_norm=w)
    # ops.rope takes its angles from a 32-bit table: off by at most 2^-24 of an angle below 64
    torch.testing.assert_close(got, ops.rope(ops.rmsnorm(q, w, 1e-6), pos, 1e6), rtol=0, atol=64 * 2.0 ** -22)


def test_append_for_more_requests_than_a_block_has_threads():
    from woodcock_b200 import ops

    B = 700
    rows = [i % 3 for i in range(B)]
    lens = [(i * 13) % 50 + r for i, r in enumerate(rows)]
    c = Case(57, lens, rows, 4, 2, 64, 16, F32)
    T = sum(rows)
    k, v = c.randn(T, 2, 64), c.randn(T, 2, 64)
    got = ops.paged_append(c.q, k, v, c.k, c.v, c.table, c.kv, q_offsets=c.off)
    b = torch.repeat_interleave(torch.arange(B, device="cuda"), i32(rows).long())
    within = torch.arange(T, device="cuda") - c.off.long()[b]
    slot = c.kv.long()[b] - i32(rows).long()[b] + within
    y, tol = want_rotated(c.q, None, slot, 1e6, 1e-6)
    assert ((got.double() - y).abs() <= tol).all()
    assert torch.equal(c.v[c.table.long()[b, slot // 16], :, slot % 16], v)


def test_append_rows_without_a_slot():
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    ctx.synchronize()
    for kv, table in (([2], [[0, 1]]), ([33], [[0, 1]]), ([20], [[0, 9]]), ([20], [[-1, 1]])):
        k = torch.full((3, 8, 16, 64), 2.0, device="cuda", dtype=BF)
        v = k.clone()
        rows = 5
        x, n = torch.randn((rows, 8, 64), device="cuda"), torch.randn((rows, 8, 64), device="cuda")
        ops.paged_append(x, n, n, k, v, i32(table[0])[None], i32(kv))
        torch.cuda.synchronize()
        with pytest.raises(WcError):
            ctx.synchronize()
        # what has a slot is written, the rest is dropped
        wrote = 0
        for i in range(rows):
            s = kv[0] - rows + i
            ok = 0 <= s < 32 and 0 <= table[0][s // 16] < 3
            wrote += ok
            if ok:
                assert torch.equal(v[table[0][s // 16], :, s % 16], n[i].to(BF))
        assert int((v != 2).any(-1).any(1).sum()) == wrote
    # rows behind the last request
    k = torch.full((3, 8, 16, 64), 2.0, device="cuda", dtype=BF)
    v, out = k.clone(), torch.full((5, 8, 64), 9.0, device="cuda", dtype=BF)
    ops.paged_append(x, n, n, k, v, i32([[0, 1]]), i32([4]), q_offsets=i32([0, 3]), out=out)
    ctx.synchronize()
    assert (out[3:] == 9).all() and int((v != 2).any(-1).any(1).sum()) == 3


# ------------------------------------------------------------------------------------------------ compaction


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("layout", ["heads", "positions"])
def test_compact(dtype, layers, layout):
    from woodcock_b200 import ops

    page, Hk, D, B = 16, 3, 64, 5
    starts = [0, 13, 16, 100, 31]
    keeps = [[0], [0, 2, 3, 9, 15, 16, 17, 30, 31, 40], [1, 2], [], [5, 20, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 32, 33, 34, 35, 36]]
    g = torch.Generator(device="cuda").manual_seed(3)
    shape = (layers, 60, Hk, page, D) if layout == "heads" else (layers, 60, page, Hk, D)
    k = torch.randn(shape, generator=g, device="cuda").to(dtype)
    v = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if layout != "heads":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    table = torch.randperm(60, generator=g, device="cuda").to(torch.int32)[:50].view(B, 10)
    m = max(map(len, keeps))
    keep = i32([x + [0] * (m - len(x)) for x in keeps])
    wk, wv = k.clone(), v.clone()
    for b in range(B):
        for want, src in ((wk, k), (wv, v)):
            for i, j in enumerate(keeps[b]):
                s, d = starts[b] + j, starts[b] + i
                want[:, table[b, d // page], :, d % page] = src[:, table[b, s // page], :, s % page]
    if layers == 1:
        lens = ops.paged_compact(k[0], v[0], table, i32(starts), keep, i32([len(x) for x in keeps]))
    else:
        lens = ops.paged_compact(k, v, table, i32(starts), keep, i32([len(x) for x in keeps]))
    assert lens.tolist() == [s + len(x) for s, x in zip(starts, keeps)]
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_compact_refuses_bad_lists_and_leaves_their_rows():
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    k = torch.randn((4, 2, 16, 64), device="cuda").to(BF)
    k0 = k.clone()
    table = i32([[0, 1], [2, 3]])
    for keep, n, starts in (([0, 0], 2, 0), ([3, 2], 2, 0), ([-1, 2], 2, 0), ([0, 40], 2, 0), ([0, 1], 3, 0), ([0, 1], -1, 0),
                            ([0, 2], 2, -1), ([0, 2 ** 31 - 1], 2, 5)):
        lens = ops.paged_compact(k, k.clone(), table, i32([starts, 3]), i32([keep, [0, 1]]), i32([n, 2]))
        torch.cuda.synchronize()
        with pytest.raises(WcError):
            ctx.synchronize()
        assert torch.equal(k, k0) and lens.tolist() == [starts, 5]
    lens = ops.paged_compact(k, k.clone(), i32([[0, 9], [2, 3]]), i32([10, 3]), i32([[0, 8], [0, 1]]), i32([2, 2]))
    torch.cuda.synchronize()
    with pytest.raises(WcError):
        ctx.synchronize()
    assert torch.equal(k, k0)
    with pytest.raises(ValueError, match="64"):
        ops.paged_compact(k, k, table, i32([0, 0]), torch.zeros((2, 65), dtype=torch.int32, device="cuda"), i32([1, 1]))


# ------------------------------------------------------------------------------------------------ use


@pytest.mark.parametrize("dtype", [BF, F32])
def test_refusals(dtype):
    from woodcock_b200 import ops

    c = Case(30, [40, 50], [1, 1], 16, 8, 128, 16, dtype)
    call = lambda **kw: ops.paged_attention(**{"q": c.q, "k_pages": c.k, "v_pages": c.v, "page_table": c.table,  # noqa: E731
                                               "kv_lens": c.kv} | kw)
    for kw in ({"q": c.q.double()}, {"q": c.q[:, :9].contiguous()}, {"q": c.q[:1].expand(3, 16, 128)}, {"kv_lens": i32([1])},
               {"q_offsets": i32([0, 2])}, {"tree_mask": i32([1, 1])}, {"scale": 0.0}, {"scale": math.inf},
               {"out": c.q[:, :8]}, {"page_table": c.table[0]}, {"scale": -1.0},
               {"tree_mask": torch.ones(3, dtype=torch.int64, device="cuda")}):
        with pytest.raises(ValueError):
            call(**kw)
    one = c.k[:1].contiguous()
    with pytest.raises(ValueError, match="overlap"):
        call(k_pages=one.expand(3, 8, 16, 128), v_pages=one.expand(3, 8, 16, 128))
    with pytest.raises(ValueError):
        ops.paged_append(c.q, c.q, c.q, c.k, c.v, c.table, c.kv)  # k has q's heads
    with pytest.raises(ValueError):
        ops.paged_append(c.q, c.q[:, :8], c.q[:, :8], c.k, c.v, c.table, c.kv, q_norm=torch.ones(64, device="cuda"))
    both = torch.zeros((5, 16, 128), dtype=dtype, device="cuda")  # an output among the inputs
    for lo in (0, 1, 2):
        with pytest.raises(ValueError, match="overlap"):
            call(q=both[1:3], out=both[lo:lo + 2])
    assert call(q=both[1:3], out=both[3:]).data_ptr() == both[3:].data_ptr()
    kv = both[3:, :8]
    for q, k, v, out in ((both[:2], kv, kv.clone(), both[1:3]), (c.q, kv, kv.clone(), both[3:]), (c.q, kv.clone(), kv, both[3:])):
        with pytest.raises(ValueError, match="overlap"):
            ops.paged_append(q, k, v, c.k.clone(), c.v.clone(), c.table, c.kv, out=out)
    with pytest.raises(ValueError, match="share"):
        ops.paged_append(c.q, kv, kv, c.k, c.k, c.table, c.kv)
    with pytest.raises(ValueError, match="share"):
        ops.paged_compact(c.k, c.k, c.table, c.kv, i32([[0], [0]]), i32([0, 0]))
    assert call(q=c.q[:0], page_table=c.table[:0], kv_lens=c.kv[:0]).shape == (0, 16, 128)
    assert call(q=c.q[:0]).shape == (0, 16, 128)


def test_threads_that_append_at_once_keep_their_own_bases():
    import threading

    from woodcock_b200 import ops

    c = Case(33, [40, 50], [1, 1], 16, 8, 128, 16, F32)
    k, v = torch.randn((2, 8, 128), device="cuda"), torch.randn((2, 8, 128), device="cuda")

    def append(base):
        return ops.paged_append(c.q, k, v, c.k.clone(), c.v.clone(), c.table, c.kv, base=base)

    want = {base: append(base) for base in (1e4, 1e6)}
    torch.cuda.synchronize()
    assert not torch.equal(want[1e4], want[1e6])
    got, errors = {1e4: [], 1e6: []}, []

    def run(base):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[base] = [append(base) for _ in range(200)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # a thread's exceptions are the test's
            errors.append(e)

    threads = [threading.Thread(target=run, args=(base,)) for base in got]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for base, outs in got.items():
        assert len(outs) == 200 and all(torch.equal(o, want[base]) for o in outs)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_steps_captured_in_graphs_follow_new_lengths_and_do_not_share_scratch(dtype):
    from woodcock_b200 import ops

    cases = [Case(31 + i, [700, 90, 300], [2, 2, 2], 16, 8, 128, 16, dtype, prefix=[100]) for i in range(2)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        call = lambda c=c: (ops.paged_attention(c.q, c.k, c.v, c.table, c.kv),  # noqa: E731
                            ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32_100, i32_03, c.table, c.kv))
        i32_100, i32_03 = i32([100]), i32([0, 3])
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            outs.append(call())
        graphs.append((g, i32_100, i32_03))
    for lens in ([700, 90, 300], [5, 2, 299], [650, 0, 17]):
        for c in cases:
            c.lens = lens
            c.kv.copy_(i32(lens))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(3):
            for s, (g, *_) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, (a, b) in zip(cases, outs):
            check(c, a)
            check(c, b, groups=[0, 3])


def test_calls_on_two_streams_at_once():
    from woodcock_b200 import ops

    a, b = Case(35, [9000, 17], [3, 3], 16, 8, 128, 16, BF), Case(36, [44, 7000], [30, 30], 16, 8, 128, 64, BF)
    want = [ops.paged_attention(c.q, c.k, c.v, c.table, c.kv) for c in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_serving_step(dtype):
    """Append, tree attention under a shared prefix, compaction of the accepted paths and the next step's
    append and attention, against one contiguous cache per request."""
    from woodcock_b200 import ops

    B, n, H, Hk, D, page, pre = 4, 7, 16, 8, 128, 16, 45
    starts = [0, 9, 16, 33]
    c = Case(40, [s + 20 for s in starts], [n] * B, H, Hk, D, page, dtype, prefix=[pre])
    w = [1 + 0.1 * torch.randn(D, generator=c.g, device="cuda") for _ in range(2)]
    bits = tree_bits([n] * B, 9)
    depth = torch.tensor([bin(x).count("1") - 1 for x in bits.tolist()], device="cuda")
    pos = torch.repeat_interleave(i32(starts), n) + depth.to(torch.int32) + pre
    proj = [c.randn(B * n, h, D) for h in (H, Hk, Hk)]
    q = ops.paged_append(*proj, c.k, c.v, c.table, i32([s + n for s in starts]), positions=pos, q_norm=w[0], k_norm=w[1])
    c.q, c.lens = q, [s + n for s in starts]
    c.kv = i32(c.lens)
    check(c, ops.shared_prefix_attention(q, c.k, c.v, c.ptable, i32([pre]), i32([0, B]), c.table, c.kv, tree_mask=bits),
          bits, [0, B])
    # accept each tree's path to its last node
    paths = [[i for i in range(n) if int(bits[b * n + n - 1]) >> i & 1] for b in range(B)]
    m = max(map(len, paths))
    flat = [[c.keys(c.k, c.table, b, c.lens[b]), c.keys(c.v, c.table, b, c.lens[b])] for b in range(B)]
    lens = ops.paged_compact(c.k, c.v, c.table, i32(starts), i32([p + [0] * (m - len(p)) for p in paths]),
                             i32([len(p) for p in paths]))
    c.lens = lens.tolist()
    assert c.lens == [s + len(p) for s, p in zip(starts, paths)]
    for b, p in enumerate(paths):
        rows = list(range(starts[b])) + [starts[b] + i for i in p]
        assert torch.equal(c.keys(c.k, c.table, b, c.lens[b]), flat[b][0][rows])
        assert torch.equal(c.keys(c.v, c.table, b, c.lens[b]), flat[b][1][rows])
    c.lens, c.rows = [x + 1 for x in c.lens], [1] * B
    c.kv = i32(c.lens)
    proj = [c.randn(B, h, D) for h in (H, Hk, Hk)]
    c.q = ops.paged_append(*proj, c.k, c.v, c.table, c.kv, positions=c.kv - 1 + pre, q_norm=w[0], k_norm=w[1])
    check(c, ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32([pre]), i32([0, B]), c.table, c.kv), groups=[0, B])
    # without a prefix this is ops.attention over the gathered rows; both round weights to bf16 at most
    out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
    for b in range(B):
        k, v = (c.keys(x, c.table, b, c.lens[b]).to(dtype) for x in (c.k, c.v))
        ref = ops.attention(c.q[b: b + 1], k, v).float()
        scale = v.float().abs().max()
        tol = 4 * half_step(BF) if dtype is BF else 2.0 ** -18
        assert (out[b: b + 1].float() - ref).abs().max() <= tol * scale
