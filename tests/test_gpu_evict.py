"""Gathered attention weight and eviction against plain implementations in 64 bits.

Tolerance of a gathered weight, for each key, relative to the formula's: a score is a sum of head_dim products in
32 bits, off by at most (head_dim + 4) 2^-24 sum |q k| scale (twice that where an adder truncates), and moves its
weight by e^x - 1; the row's sum moves by as much the other way; 2^-19 covers the exponentials, the scale and the
maximum (|s| < 64, log2 units), (keys + rows) 2^-24 the sums. What was there before is added with one rounding.
Eviction moves bits.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged import BF, F32, Case, half_step, i32, offsets, want_rows

pytestmark = pytest.mark.gpu


def mass_of(c, fill=None):
    """Mass pages beside a case's pages: random, NaN where no key lies."""
    total, Hk, page = c.k.shape[:3]
    m = torch.full((total, Hk, page), math.nan, device="cuda")
    for b, n in enumerate(c.lens):
        at = torch.arange(n, device="cuda")
        m[c.table[b].long()[at // page], :, at % page] = torch.rand((n, Hk), generator=c.g, device="cuda") * 3
    return m if fill is None else m.fill_(fill)


def at_keys(pool, c, b, n):
    at = torch.arange(n, device="cuda")
    return pool[c.table[b].long()[at // c.page], :, at % c.page]


def gathered(c, b, t0, scale=None):
    """[n][Hk]: the formula in 64 bits for request b, and the bound of its relative error."""
    n, r, rep = c.lens[b], c.rows[b], c.H // c.Hk
    k = c.keys(c.k, c.table, b, n).repeat_interleave(rep, 1)
    q = c.q[t0: t0 + r].double()
    scale = c.D ** -0.5 if scale is None else scale
    sees = torch.arange(n, device="cuda")[None] <= torch.arange(n - r, n, device="cuda")[:, None]
    out, worst = torch.zeros((n, c.Hk), dtype=torch.float64, device="cuda"), 0.0
    for h in range(c.H):
        s = (q[:, h] @ k[:, h].T) * scale
        p = torch.softmax(torch.where(sees, s, -math.inf), -1)
        out[:, h // rep] += torch.where(sees.any(1, keepdim=True), p, 0.0).sum(0)
        worst = max(worst, float((q[:, h].abs() @ k[:, h].abs().T).max()) * scale if n else 0.0)
    es = 2 * (c.D + 4) * 2.0 ** -24 * worst
    return out, 2 * math.expm1(es) + 2.0 ** -19 + (n + r * rep) * 2.0 ** -24


def check(c, before, after, add=True, scale=None):
    t0 = 0
    touched = torch.zeros(after.shape, dtype=torch.bool, device="cuda")
    for b, (n, r) in enumerate(zip(c.lens, c.rows)):
        if n and r:
            want, rel = gathered(c, b, t0, scale)
            was = at_keys(before, c, b, n).double().clone()
            was[max(0, n - r) if add else 0:] = 0
            got = at_keys(after, c, b, n).double()
            tol = want * rel + (was + want) * 2.0 ** -23
            assert torch.isfinite(got).all(), f"request {b}"
            over = ((got - was - want).abs() - tol).max()
            assert over <= 0, f"request {b}: {float(over)} over"
            at = torch.arange(n, device="cuda")
            touched[c.table[b].long()[at // c.page], :, at % c.page] = True
        t0 += r
    same = (after == before) | (after.isnan() & before.isnan())
    assert bool((same | touched).all()), "written where no key lies"


@pytest.mark.parametrize("H, Hk, D, page, dtype, rows, lens", [
    (16, 8, 128, 16, BF, [1], [1]),
    (16, 8, 128, 16, BF, [1], [513]),
    (32, 8, 128, 64, BF, [1, 1, 1], [63, 64, 65]),
    (8, 1, 64, 16, BF, [1, 1], [2000, 3]),                  # eight heads on one key head
    (40, 8, 128, 32, BF, [2, 3, 1, 3], [17, 900, 0, 128]),  # an idle slot; 15 rows a head at most
    (6, 2, 64, 128, F32, [5, 5], [600, 129]),
    (4, 2, 64, 16, F32, [1, 40, 7], [100, 41, 7]),
    (4, 4, 128, 256, F32, [3], [1000]),
    (16, 8, 128, 16, BF, [9, 8, 1], [40, 300, 5]),          # 16 and 18 rows a head
    (32, 8, 128, 64, BF, [32, 32], [1500, 33]),             # a window: 128 rows a head
    (32, 8, 64, 16, BF, [33, 7, 20], [500, 7, 1000]),
    (8, 8, 128, 128, BF, [130, 1], [130, 70]),              # a prompt beside a step
    (12, 4, 64, 32, BF, [300, 171], [300, 700]),
    (5, 1, 128, 16, BF, [77, 100], [64, 1000]),             # more rows than keys: the first see nothing
    (4, 1, 128, 64, BF, [700], [2500]),
])
@pytest.mark.parametrize("add", [True, False])
def test_gathered_weight(H, Hk, D, page, dtype, rows, lens, add):
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    c = Case(1, lens, rows, H, Hk, D, page, dtype)
    before = mass_of(c)
    for b, (n, r) in enumerate(zip(lens, rows)):  # what a new key's place held before does not count
        at = torch.arange(max(0, n - r) if add else 0, n, device="cuda")
        before[c.table[b].long()[at // page], :, at % page] = math.nan
    mass = before.clone()
    assert ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off, add=add) is mass
    Context.get(0).synchronize()
    check(c, before, mass, add)


@pytest.mark.parametrize("rows, lens", [([1] * 300, [(i * 37) % 90 for i in range(300)]),
                                        ([1 + i % 3 for i in range(130)], [3 + (i * 53) % 200 for i in range(130)]),
                                        ([(i * 7) % 40 for i in range(90)], [40 + (i * 53) % 200 for i in range(90)])])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_requests(rows, lens, dtype):
    from woodcock_b200 import ops

    c = Case(2, lens, rows, 8, 2, 64, 16, dtype)
    before = mass_of(c)
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off)
    check(c, before, mass)
    again = before.clone()
    ops.paged_mass(c.q, c.k, again, c.table, c.kv, q_offsets=c.off)
    assert torch.equal(mass.nan_to_num(-1), again.nan_to_num(-1))


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_scale_and_rows_behind_the_last(rows, dtype):
    from woodcock_b200 import ops

    c = Case(3, [70, 300], [rows, rows], 16, 8, 128, 32, dtype, layout="rows")
    fused = torch.full((2 * rows + 5, 40, 128), math.nan, dtype=dtype, device="cuda")
    fused[: 2 * rows, 3:19] = c.q
    q = fused[:, 3:19]  # a projection's columns, and rows that belong to nobody
    total = c.k.shape[0]
    wide = torch.full((total, 3, 8, 32), math.nan, device="cuda")
    mass = wide[:, 1]
    mass.copy_(mass_of(c))
    before = mass.clone()
    ops.paged_mass(q, c.k, mass, c.table, c.kv, q_offsets=offsets([rows, rows]), scale=0.3)
    check(c, before, mass, scale=0.3)
    assert wide[:, 0].isnan().all() and wide[:, 2].isnan().all()


@pytest.mark.parametrize("rows", [1, 30])
def test_a_row_beside_what_is_not_finite(rows):
    """A key that is NaN makes the weights of the rows that see it NaN, and of no others."""
    from woodcock_b200 import ops

    c = Case(4, [200, 200], [rows, rows], 16, 8, 128, 16, BF)
    page, r = c.table[0, 199 // 16].long(), 199 % 16
    c.k[page, 3, r] = math.nan  # the last key of one head: its request's last row sees it
    before = mass_of(c, 0.5)
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv)
    got = at_keys(mass, c, 0, 200)
    assert got[:, 3].isnan().all()
    assert torch.isfinite(got[:, [0, 1, 2, 4, 5, 6, 7]]).all() and torch.isfinite(at_keys(mass, c, 1, 200)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows, lens", [
    ([0, 1, 0, 2, 0], [700, 90, 0, 33, 64]),                # idle requests among steps
    ([40, 0, 1, 0], [200, 333, 70, 5]),                     # beside a window
    ([0] * 3, [257, 0, 1]),                                 # nobody has a row, offsets say so
    ([0, 3] * 200, [(i * 37) % 90 for i in range(400)]),    # more requests than blocks
])
def test_requests_without_rows_start_anew_too(dtype, rows, lens):
    """add=False: every key's sum is that of this call's weights, 0 where no row looks; with add nothing changes."""
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    c = Case(21, lens, rows, 8, 2, 64, 16, dtype)
    before = mass_of(c)
    for b, n in enumerate(lens):  # what lies there does not count
        at = torch.arange(n, device="cuda")
        before[c.table[b].long()[at // 16], :, at % 16] = math.nan
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off, add=False)
    Context.get(0).synchronize()
    idle = before.clone()
    for b, (n, r) in enumerate(zip(lens, rows)):
        if r == 0:
            assert (at_keys(mass, c, b, n) == 0).all(), f"request {b}"
            at = torch.arange(n, device="cuda")
            idle[c.table[b].long()[at // 16], :, at % 16] = 0.0
    check(c, idle, mass, add=False)
    before = mass_of(c)
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off)
    check(c, before, mass)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_call_without_rows_or_offsets(dtype):
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    c = Case(22, [100, 17], [0, 0], 4, 2, 64, 32, dtype, layout="rows")
    before = mass_of(c)
    mass = before.clone()
    assert ops.paged_mass(c.q, c.k, mass, c.table, c.kv) is mass
    assert torch.equal(mass.nan_to_num(-1), before.nan_to_num(-1))
    assert ops.paged_mass(c.q, c.k, mass, c.table, c.kv, add=False) is mass
    want = before.clone()
    for b, n in enumerate(c.lens):
        at = torch.arange(n, device="cuda")
        want[c.table[b].long()[at // 32], :, at % 32] = 0.0
    assert torch.equal(mass.nan_to_num(-1), want.nan_to_num(-1))
    Context.get(0).synchronize()
    for kw, what in (({"mass_pages": mass.double()}, "fp32"), ({"scale": -1.0}, "scale"),
                     ({"mass_pages": mass[:1].expand(mass.shape)}, "overlap")):
        with pytest.raises(ValueError, match=what):  # refused as with rows
            ops.paged_mass(**{"q": c.q, "k_pages": c.k, "mass_pages": mass, "page_table": c.table, "kv_lens": c.kv, "add": False, **kw})
    table = c.table.clone()
    table[0, 1] = -1
    ops.paged_mass(c.q, c.k, mass, table, c.kv, add=False)
    with pytest.raises(WcError):
        Context.get(0).synchronize()


@pytest.mark.parametrize("rows, H, dtype", [(5, 8, BF), (2, 32, BF), (5, 8, F32), (40, 8, BF), (200, 8, BF)])
@pytest.mark.parametrize("first", [0, 1])
def test_a_row_that_is_not_finite_weighs_what_it_sees(rows, H, dtype, first):
    """A NaN in a row's query makes the keys NaN that the row sees; those behind them keep the other rows' weight."""
    from woodcock_b200 import ops

    c = Case(23, [100, 300], [rows, rows], H, 4, 64, 16, dtype)
    rep, clean = H // 4, c.q.clone()
    c.q[first, 2 * rep] = math.nan  # of the first request, third key head
    before = mass_of(c, 0.5)
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv)
    seen = max(0, 100 - rows + first + 1)
    got = at_keys(mass, c, 0, 100)
    assert got[:seen, 2].isnan().all()
    c.q = clean
    c.q[first] = 0  # the formula without the row's weight: at the keys it does not see it has none
    want, rel = gathered(c, 0, 0)
    late = got[seen:, 2].double()
    assert ((late - want[seen:, 2]).abs() <= want[seen:, 2] * (rel + 2.0 ** -23)).all()
    assert torch.isfinite(got[:, [0, 1, 3]]).all() and torch.isfinite(at_keys(mass, c, 1, 300)).all()


@pytest.mark.parametrize("rows, dtype", [(1, BF), (5, BF), (5, F32), (20, BF), (40, BF), (150, BF)])
def test_a_key_that_no_row_can_want(rows, dtype):
    """A key that is -inf where every query is positive has the score -inf: no weight, and none lost by the others."""
    from woodcock_b200 import ops

    c = Case(24, [200, 333], [rows, rows], 8, 4, 64, 16, dtype)
    c.q[:, :, 5] = c.q[:, :, 5].abs() + 0.5
    want, rel = [], []
    for b in range(2):  # the formula with a key far away, whose weight is 0 in 64 bits
        c.k[c.table[b, 2].long(), 1, 3] = 0.0
        c.k[c.table[b, 2].long(), 1, 3, 5] = -3e4
        w, _ = gathered(c, b, b * rows)
        assert w[35, 1] == 0
        want.append(w)
        c.k[c.table[b, 2].long(), 1, 3, 5] = 0.0
        rel.append(gathered(c, b, b * rows)[1])  # the bound is of the other keys' scores
        c.k[c.table[b, 2].long(), 1, 3, 5] = -math.inf
    mass = mass_of(c, math.nan)
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, add=False)
    for b in range(2):
        got = at_keys(mass, c, b, c.lens[b]).double()
        assert torch.isfinite(got).all()
        assert ((got - want[b]).abs() <= want[b] * (rel[b] + 2.0 ** -23)).all()


@pytest.mark.parametrize("rows, dtype", [(1, BF), (20, BF), (3, F32)])
def test_bad_tables_raise_the_error_word(rows, dtype):
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    c = Case(5, [100, 50], [rows, rows], 8, 4, 64, 16, dtype)
    ctx = Context.get(0)
    ctx.synchronize()
    before = mass_of(c)
    for page, lens in ((c.k.shape[0], c.kv), (-1, c.kv), (None, i32([100, 113])), (None, i32([-4, 50]))):
        table, mass = c.table.clone(), before.clone()
        if page is not None:
            table[1, 1] = page
        ops.paged_mass(c.q, c.k, mass, table, lens)
        with pytest.raises(WcError):
            ctx.synchronize()
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv)
    ctx.synchronize()
    check(c, before, mass)


def test_requests_that_share_pages_leave_the_mass_as_it_was():
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    c = Case(6, [320], [1], 8, 4, 64, 16, BF)
    ctx = Context.get(0)
    ctx.synchronize()
    table = c.table.expand(64, -1).contiguous()
    q = c.q.expand(64, -1, -1).contiguous()
    before = mass_of(c)
    mass = before.clone()
    ops.paged_mass(q, c.k, mass, table, c.kv.expand(64).contiguous())
    with pytest.raises(WcError):
        ctx.synchronize()
    assert torch.equal(mass.nan_to_num(-1), before.nan_to_num(-1))


@pytest.mark.parametrize("rows, dtype", [([1, 1], BF), ([5, 5], BF), ([20, 20], BF), ([200, 200], BF), ([3, 3], F32), ([1, 20], BF),
                                         ([40, 0], BF), ([0, 3], F32)])
def test_more_pages_than_the_pool_has_raise_the_error_word(rows, dtype):
    """Two requests on the same 20 pages of 21, whichever kernels their rows take; a pool that is full to its last page will do."""
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    ctx.synchronize()
    c = Case(25, [320], [sum(rows)], 8, 4, 64, 16, dtype)
    ops.paged_mass(c.q, c.k, mass_of(c, 0.0), c.table.expand(2, -1).contiguous(), i32([320, 320]), q_offsets=offsets(rows),
                   add=False)
    with pytest.raises(WcError):
        ctx.synchronize()
    c = Case(25, [320, 161], rows, 8, 4, 64, 16, dtype, spare=0)
    for b in range(2):  # every page of the pool
        c.lens[b] = 320
    c.kv = i32(c.lens)
    c.k.nan_to_num_(0.25)
    before = mass_of(c)
    mass = before.clone()
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off)
    ctx.synchronize()
    check(c, before, mass)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_requests_that_fall_idle_between_replays(dtype):
    """Offsets are device data: a captured call that starts the sums anew meets requests without rows at a replay."""
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    c = Case(26, [300, 90, 41], [2, 30, 4], 8, 2, 64, 16, dtype)
    mass = mass_of(c, math.nan)
    ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off, add=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off, add=False)
    for rows in ([0, 30, 6], [36, 0, 0], [0, 0, 0], [2, 30, 4]):
        c.rows = rows
        c.off.copy_(offsets(rows))
        mass.fill_(math.nan)
        graph.replay()
        before = torch.full_like(mass, math.nan)
        for b, (n, r) in enumerate(zip(c.lens, rows)):
            if r == 0:
                assert (at_keys(mass, c, b, n) == 0).all()
                at = torch.arange(n, device="cuda")
                before[c.table[b].long()[at // 16], :, at % 16] = 0.0
        check(c, before, mass, add=False)
    Context.get(0).synchronize()


def test_arguments_of_mass_that_are_refused():
    from woodcock_b200 import ops

    c = Case(7, [40, 50], [1, 1], 16, 8, 128, 16, BF)
    mass = mass_of(c)
    for kw, what in (({"mass_pages": mass.double()}, "fp32"), ({"mass_pages": mass[:-1]}, "fp32"),
                     ({"mass_pages": mass.transpose(1, 2).contiguous().transpose(1, 2)}, "contiguous"),
                     ({"mass_pages": mass.cpu()}, "fp32"), ({"q": c.q.float()}, "must be"), ({"q": c.q[:, :12]}, "multiple"),
                     ({"q": c.q[:, :, :64]}, "must be"), ({"kv_lens": i32([1])}, "entries"), ({"scale": -1.0}, "scale"),
                     ({"scale": math.nan}, "scale"), ({"q_offsets": i32([0, 2])}, "entries"),
                     ({"mass_pages": mass[:1].expand(mass.shape)}, "overlap"),
                     ({"mass_pages": torch.as_strided(mass, mass.shape, (64, 16, 1))}, "overlap"),
                     ({"mass_pages": c.k.view(torch.float32).view(-1)[: mass.numel()].view(mass.shape)}, "overlap")):
        args = {"q": c.q, "k_pages": c.k, "mass_pages": mass, "page_table": c.table, "kv_lens": c.kv, **kw}
        with pytest.raises(ValueError, match=what):
            ops.paged_mass(**args)
    inside = c.kv.new_zeros(mass.numel()).view(torch.float32).view(mass.shape)
    with pytest.raises(ValueError, match="overlap"):  # lengths inside the mass
        ops.paged_mass(c.q, c.k, inside, c.table, inside.view(torch.int32).view(-1)[:2])


# ---------------------------------------------------------------------------- eviction


class Pool:
    """Every layer's pages with scattered tables; what holds no key is marked."""

    def __init__(self, seed, lens, L, Hk, D, page, dtype, spare=2, quant=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.L, self.Hk = lens, page, L, Hk
        width = max(1, max(-(-n // page) for n in lens))
        total = len(lens) * width + spare
        self.table = torch.randperm(total, generator=g, device="cuda")[: len(lens) * width].view(len(lens), width).to(torch.int32)
        self.k = torch.randn((L, total, Hk, page, D), generator=g, device="cuda").to(dtype)
        self.v = torch.randn((L, total, Hk, page, D), generator=g, device="cuda").to(dtype)
        self.mass = torch.randn((L, total, Hk, page), generator=g, device="cuda")
        if quant:
            self.mass = (self.mass * quant).round() / quant
        self.kv = i32(lens)

    def where(self, b, keys):
        return self.table[b].long()[keys // self.page], keys % self.page


def evicted(c, budgets, sinks, recent):
    """The formula: k, v, mass and lengths."""
    k, v, mass, lens = c.k.clone(), c.v.clone(), c.mass.clone(), list(c.lens)
    for b, (n, m) in enumerate(zip(c.lens, budgets)):
        if n <= m or m < sinks + recent:
            continue
        lens[b] = m
        every = torch.arange(n, device="cuda")
        ps, rs = c.where(b, every)
        pd, rd = c.where(b, every[:m])
        for layer in range(c.L):
            for h in range(c.Hk):
                w = c.mass[layer, ps, h, rs].double()
                middle = torch.where(w.isnan(), -math.inf, w)[sinks: n - recent]
                # NaN below -inf: rank by (is a number, value), ties to the lower key
                order = sorted(range(n - recent - sinks), key=lambda j, m=middle.tolist(), w=w[sinks:].tolist():
                               (math.isnan(w[j]), -m[j], j)) if w.isnan().any() else \
                    torch.argsort(middle, descending=True, stable=True).tolist()
                keep = sorted([*range(sinks), *(sinks + j for j in order[: m - sinks - recent]), *range(n - recent, n)])
                kept = torch.tensor(keep, dtype=torch.int64, device="cuda")
                for x, src in ((k, c.k), (v, c.v), (mass, c.mass)):
                    x[layer, pd, h, rd] = src[layer, ps[kept], h, rs[kept]]
    return k, v, mass, lens


def bits(x):
    return x.view(torch.int16 if x.element_size() == 2 else torch.int32)


def check_evict(c, budgets, sinks, recent, arg=None):
    from woodcock_b200 import ops

    k, v, mass, lens = evicted(c, budgets, sinks, recent)
    got = ops.paged_evict(c.k, c.v, c.mass, c.table, c.kv, budgets[0] if arg is None else arg, sinks=sinks, recent=recent)
    assert got.tolist() == lens and got.dtype is torch.int32
    for x, y in ((c.k, k), (c.v, v), (c.mass, mass)):
        assert torch.equal(bits(x), bits(y))


@pytest.mark.parametrize("lens, L, Hk, D, page, dtype, budget, sinks, recent", [
    ([2], 1, 1, 64, 16, BF, 1, 0, 0),
    ([1, 5], 2, 2, 128, 16, BF, 0, 0, 0),                  # nothing stays
    ([640], 3, 8, 128, 16, BF, 512, 4, 64),
    ([513, 100, 512, 0, 514], 2, 4, 64, 32, F32, 512, 4, 64),
    ([513], 2, 4, 128, 128, F32, 512, 0, 512),             # the first goes
    ([700], 1, 2, 64, 64, BF, 100, 100, 0),                # the first ones stay
    ([700], 1, 2, 64, 64, BF, 100, 40, 60),                # nothing to choose
    ([300, 1000, 77], 2, 3, 128, 256, BF, 65, 1, 7),
    ([20000, 16400], 1, 2, 64, 64, BF, 3001, 4, 100),      # more sums than shared memory holds
    ([1025], 2, 2, 128, 16, BF, 1024, 0, 0),
    # lists enough that one kernel selects and moves
    ([300, 1, 700, 333, 65], 8, 4, 128, 32, BF, 64, 2, 9),
    ([17000, 16384, 900], 10, 5, 64, 16, BF, 900, 3, 50),
    ([129] * 40, 1, 4, 64, 128, F32, 128, 0, 1),
])
def test_eviction(lens, L, Hk, D, page, dtype, budget, sinks, recent):
    check_evict(Pool(8, lens, L, Hk, D, page, dtype), [budget] * len(lens), sinks, recent)


@pytest.mark.parametrize("quant", [0.001, 1, 4])  # all alike, a handful of values, many ties
def test_ties_stay_with_the_lower_key(quant):
    check_evict(Pool(9, [700, 1300], 2, 2, 64, 16, BF, quant=quant), [300, 300], 5, 11)


def test_masses_that_are_no_numbers():
    c = Pool(10, [400, 90], 1, 2, 64, 16, BF)
    g = torch.Generator(device="cuda").manual_seed(1)
    r = torch.rand(c.mass.shape, generator=g, device="cuda")
    c.mass[r < 0.7] = math.nan
    c.mass[(r > 0.70) & (r < 0.75)] = math.inf
    c.mass[(r > 0.75) & (r < 0.80)] = -math.inf
    c.mass[(r > 0.80) & (r < 0.85)] = 0.0
    c.mass[(r > 0.85) & (r < 0.90)] = -0.0
    check_evict(c, [200, 50], 2, 3, arg=i32([200, 50]))


def test_budgets_of_their_own():
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    Context.get(0).synchronize()
    budgets = [100, 300, 20, 64, 7]
    check_evict(Pool(11, [250, 250, 64, 64, 250], 2, 2, 64, 16, BF), budgets, 3, 4, arg=i32(budgets))
    Context.get(0).synchronize()
    c = Pool(11, [250, 250], 2, 2, 64, 16, BF)
    check_evict(c, [6, 100], 3, 4, arg=i32([6, 100]))  # the first is below what is protected: it stays as it is
    with pytest.raises(WcError):
        Context.get(0).synchronize()


def test_strided_pages_and_k_and_v_in_one_buffer():
    from woodcock_b200 import ops

    c = Pool(12, [200, 130], 3, 4, 64, 16, BF)
    k, v, mass, lens = evicted(c, [90, 90], 2, 20)
    total = c.k.shape[1]
    both = torch.zeros((total, 3, 16, 4, 2, 64), dtype=BF, device="cuda")  # pages, layers, rows, heads, K and V
    kk, vv = (both[:, :, :, :, i].permute(1, 0, 3, 2, 4) for i in range(2))
    mm = torch.zeros((total, 4, 3, 16), device="cuda").permute(2, 0, 1, 3)
    kk.copy_(c.k), vv.copy_(c.v), mm.copy_(c.mass)
    assert ops.paged_evict(kk, vv, mm, c.table, c.kv, 90, sinks=2, recent=20).tolist() == lens
    assert torch.equal(kk, k) and torch.equal(vv, v) and torch.equal(mm, mass)


def test_bad_requests_keep_their_rows():
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    Context.get(0).synchronize()
    c = Pool(13, [200, 130, 150], 2, 2, 64, 16, BF)
    c.lens = [200, 0, 0]
    k, v, mass, _ = evicted(c, [90, 90, 90], 2, 20)
    table = c.table.clone()
    table[1, 4] = c.k.shape[1]
    lens = i32([200, 130, c.table.shape[1] * 16 + 1])
    got = ops.paged_evict(c.k, c.v, c.mass, table, lens, 90, sinks=2, recent=20)
    with pytest.raises(WcError):
        Context.get(0).synchronize()
    assert got.tolist() == [90, 130, c.table.shape[1] * 16 + 1]
    assert torch.equal(c.k, k) and torch.equal(c.v, v) and torch.equal(c.mass, mass)


def test_arguments_of_evict_that_are_refused():
    from woodcock_b200 import ops

    c = Pool(14, [40, 50], 2, 2, 64, 16, BF)
    for kw, what in (({"budget": 5, "sinks": 3, "recent": 3}, "budget"), ({"budget": -1}, "budget"), ({"sinks": -1}, "negative"),
                     ({"recent": -1}, "negative"), ({"budget": i32([1])}, "entries"), ({"mass_pages": c.mass[0]}, "fp32"),
                     ({"v_pages": c.k}, "share"), ({"kv_lens": i32([1])}, "entries"), ({"k_pages": c.k[0]}, "alike"),
                     ({"mass_pages": c.mass[:1].expand(c.mass.shape)}, "overlap"),
                     ({"mass_pages": c.v.view(torch.float32).view(-1)[: c.mass.numel()].view(c.mass.shape)}, "overlap"),
                     ({"kv_lens": c.mass.view(torch.int32).view(-1)[:2]}, "overlap"),
                     ({"budget": c.k.view(torch.int32).view(-1)[:2]}, "overlap")):
        args = {"k_pages": c.k, "v_pages": c.v, "mass_pages": c.mass, "page_table": c.table, "kv_lens": c.kv, "budget": 20, **kw}
        with pytest.raises(ValueError, match=what):
            ops.paged_evict(**args)


def test_captured_and_replayed_on_new_lengths():
    from woodcock_b200 import ops

    c = Case(15, [300, 40], [1, 1], 16, 8, 128, 16, BF)
    v = torch.randn(c.k.shape, generator=c.g, device="cuda").to(BF)
    first = mass_of(c, 0.25)
    k0, v0 = c.k.clone(), v.clone()

    def call(k, vv, mass, lens):
        ops.paged_mass(c.q, k, mass, c.table, lens)
        return ops.paged_evict(k, vv, mass, c.table, lens, 64, sinks=2, recent=8)

    lens = i32([300, 40])
    k, vv, mass = k0.clone(), v0.clone(), first.clone()
    call(k, vv, mass, lens)  # before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(k, vv, mass, lens)
    for n in ([300, 40], [129, 40], [65, 33], [300, 0]):
        k.copy_(k0), vv.copy_(v0), mass.copy_(first), lens.copy_(i32(n))
        graph.replay()
        want = (k0.clone(), v0.clone(), first.clone())
        got = call(*want, i32(n))
        assert out.tolist() == got.tolist() == [min(x, 64) for x in n]
        for x, y in zip((k, vv, mass), want):
            assert torch.equal(bits(x), bits(y))


def test_other_streams_and_two_at_once():
    from woodcock_b200 import ops

    cases = [Case(16 + i, [900, 300 + i], [r, r], 16, 8, 128, 16, BF) for i, r in enumerate((1, 12, 1, 12))]
    masses = [mass_of(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [m.clone() for m in masses]
    torch.cuda.synchronize()
    for _ in range(3):
        for m, g in zip(masses, got):
            g.copy_(m)
        torch.cuda.synchronize()
        for c, g, s in zip(cases, got, streams):
            with torch.cuda.stream(s):
                ops.paged_mass(c.q, c.k, g, c.table, c.kv)
        torch.cuda.synchronize()
        for c, m, g in zip(cases, masses, got):
            check(c, m, g)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_far_into_a_large_pool(rows):
    """Offsets beyond 2^31 elements: K, V and their sums."""
    from woodcock_b200 import ops

    total, cols = 140_000, 10  # 16384 elements a page
    c = Case(17, [150], [rows], 16, 8, 128, 16, BF, spare=0)
    far = torch.randperm(cols, generator=c.g, device="cuda") + total - cols
    k, v = (torch.empty((total, 8, 16, 128), dtype=BF, device="cuda") for _ in range(2))
    mass = torch.empty((total, 8, 16), device="cuda")
    near = mass_of(c)
    order = c.table[0].long()
    k[far], v[far], mass[far] = c.k[order], c.v[order], near[order]
    table = far.to(torch.int32)[None].contiguous()
    ops.paged_mass(c.q, k, mass, table, c.kv)
    after = near.clone()
    after[order] = mass[far]
    check(c, near, after)
    p = Pool.__new__(Pool)
    p.k, p.v, p.mass, p.lens, p.page, p.L, p.Hk, p.table = k[far][None].clone(), v[far][None].clone(), mass[far][None].clone(), [150], 16, \
        1, 8, torch.arange(cols, device="cuda", dtype=torch.int32)[None]
    want = evicted(p, [70], 3, 9)
    assert ops.paged_evict(k, v, mass, table, c.kv, 70, sinks=3, recent=9).tolist() == [70]
    for x, y in ((k, want[0]), (v, want[1]), (mass, want[2])):
        assert torch.equal(bits(x[far]), bits(y[0]))


# ---------------------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_session_within_its_budget(dtype):
    """A prompt, then steps and accepted chains; whenever the keys outgrow the budget they are evicted. After every
    call what the pages hold is what the formulas make of what they held: heads keep keys of their own, attention
    and gathered weights go over those."""
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    H, Hk, D, page, B, budget, sinks, recent = 8, 4, 64, 16, 2, 48, 2, 8
    c = Case(20, [0] * B, [1] * B, H, Hk, D, page, dtype, spare=B * 6)
    c.table = torch.randperm(c.k.shape[0], generator=c.g, device="cuda")[: B * 6].view(B, 6).to(torch.int32)
    mass = torch.full(c.k.shape[:3], math.nan, device="cuda")
    h = half_step(dtype)
    seen, evictions = [0] * B, 0
    for rows in ([60, 70], [1, 1], [5, 2], [1, 1], [1, 1], [5, 4], [5, 5], [5, 1], [1, 1]):
        T = sum(rows)
        kn, vn = (c.randn(T, Hk, D) for _ in range(2))
        pos = i32([seen[b] + i for b in range(B) for i in range(rows[b])])
        c.rows, c.lens = rows, [n + r for n, r in zip(c.lens, rows)]
        c.kv, c.off = i32(c.lens), offsets(rows)
        c.q = ops.paged_append(c.randn(T, H, D, scale=1.5), kn, vn, c.k, c.v, c.table, c.kv, positions=pos, q_offsets=c.off)
        out = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off).double()
        t0 = 0
        for b in range(B):
            o, a, es = want_rows(c, b, t0)[:3]
            tol = (h if dtype is BF else 0) * (o.abs() + a) + (2 * es + c.lens[b] * 2.0 ** -24 + 2.0 ** -12) * a
            assert ((out[t0: t0 + rows[b]] - o).abs() <= tol).all()
            t0 += rows[b]
        before = mass.clone()
        ops.paged_mass(c.q, c.k, mass, c.table, c.kv, q_offsets=c.off)
        check(c, before, mass)
        p = Pool.__new__(Pool)
        p.k, p.v, p.mass = c.k[None].clone(), c.v[None].clone(), mass[None].clone()
        p.lens, p.page, p.L, p.Hk, p.table = c.lens, page, 1, Hk, c.table
        k, v, m, lens = evicted(p, [budget] * B, sinks, recent)
        evictions += sum(n > budget for n in c.lens)
        assert ops.paged_evict(c.k, c.v, mass, c.table, c.kv, budget, sinks=sinks, recent=recent).tolist() == lens
        for x, y in ((c.k, k[0]), (c.v, v[0]), (mass, m[0])):
            assert torch.equal(bits(x), bits(y))
        c.lens = lens
        seen = [s + r for s, r in zip(seen, rows)]
    assert evictions >= 8
    Context.get(0).synchronize()
