"""Beam selection and reordering against plain implementations.

Tolerances. Ranks, parents and tokens are equal to those of the formula in 64 bits wherever neighbours in rank are
further apart than the sum of exponentials can be off: each term is off by at most 2^-22 and its 32-bit sum
over at most 32 values by 2^-19, so log-sum-exp by 2^-18; the inputs here (checked) keep 2^-16 between the ranks that
matter, unless they tie exactly. A score is given in 32 bits: 2^-24 of it, and the log-sum-exp's 2^-18.
Reordering moves bits.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged import BF, F32, i32

pytestmark = pytest.mark.gpu

GAP, LSE = 2.0 ** -16, 2.0 ** -18


def selected(logits, scores, n, finished=None, pad=0):
    """The formula: (scores in 64 bits, parents, tokens), and whether ranks are apart or tied exactly."""
    B, W, V = logits.shape
    z = logits.double().cpu()
    out, apart = [], True
    for b in range(B):
        cand = []
        for w in range(W):
            s = float(scores[b, w])
            if not -math.inf < s < math.inf:
                continue
            if finished is not None and bool(finished[b, w]):
                cand.append((-s, w, pad))
                continue
            row = z[b, w]
            if row.isnan().any() or (row == math.inf).any() or (row == -math.inf).all():
                continue
            score = s + (row - torch.logsumexp(row, 0))
            top = torch.argsort(score, descending=True, stable=True)[: n + 1].tolist()
            cand += [(-float(score[t]), w, t) for t in top if score[t] > -math.inf]
        cand.sort()
        for x, y in zip(cand[:n], cand[1: n + 1]):
            gap = y[0] - x[0]
            apart &= gap > GAP or (gap == 0 and x[1] == y[1]) or (gap == 0 and torch.equal(z[b, x[1]], z[b, y[1]]))
        cand = cand[:n] + [(math.inf, 0, 0)] * (n - len(cand[:n]))
        out.append(cand)
    return (torch.tensor([[-c[0] for c in r] for r in out], dtype=torch.float64), torch.tensor([[c[1] for c in r] for r in out]),
            torch.tensor([[c[2] for c in r] for r in out]), apart)


def check(logits, scores, n, finished=None, pad=0, apart=True):
    from woodcock_b200 import ops

    want = selected(logits, scores, n, finished, pad)
    assert want[3] or not apart, "the inputs' ranks are too close to tell"
    got = ops.beam_select(logits, scores, n, finished=finished, pad=pad)
    for x in got:
        assert x.shape == (logits.shape[0], n)
    g, w = got[0].double().cpu(), want[0]
    assert torch.equal(g == -math.inf, w == -math.inf)
    real = w > -math.inf
    assert ((g - w).abs()[real] <= w.abs()[real] * 2.0 ** -24 + LSE).all()
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
    return got


def spaced(seed, B, W, V, dtype=F32):
    """Logits whose best ones are well apart, and scores."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn((B, W, V), generator=g, device="cuda") * 2.5
    return z.to(dtype), -(5 + 3 * torch.rand((B, W), generator=g, device="cuda"))


def try_seeds(B, W, V, n, dtype=F32, **kw):
    """The first of a few seeds whose ranks are apart."""
    for seed in range(20):
        z, s = spaced(seed, B, W, V, dtype)
        if selected(z, s, n, **kw)[3]:
            return z, s
    raise AssertionError("no seed keeps the ranks apart")


@pytest.mark.parametrize("B, W, V, n", [
    (1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 2, 6), (1, 1, 7, 7), (3, 2, 50, 64), (1, 4, 4099, 8), (2, 5, 8192, 5), (1, 3, 8193, 12),
    (1, 2, 8186, 4), (5, 1, 16385, 3), (1, 64, 1000, 64), (2, 33, 300, 33), (1, 4, 151936, 8), (70, 2, 129, 4), (1, 1, 40000, 64),
])
def test_selection(B, W, V, n):
    check(*try_seeds(B, W, V, n), n)


@pytest.mark.parametrize("B, W, V, n", [(2, 3, 501, 6), (1, 4, 16384, 16), (3, 8, 8200, 16), (1, 32, 2000, 64)])
def test_selection_of_bf16_logits(B, W, V, n):
    """bf16 logits tie within a beam: the lower token comes first."""
    for seed in range(40):
        z, s = spaced(seed, B, W, V, BF)
        if selected(z, s, n)[3]:
            break
    check(z, s, n)


@pytest.mark.parametrize("dtype, V, shift", [(F32, 1001, 1), (F32, 8191, 3), (BF, 1001, 1), (BF, 8190, 5), (BF, 20001, 7)])
def test_rows_that_begin_anywhere(dtype, V, shift):
    """Views of a wider head's logits: rows begin off every boundary, and what lies beside them does not count."""
    z, s = try_seeds(2, 3, V, 6, dtype)
    wide = torch.full((2, 5, V + 29), math.nan, dtype=dtype, device="cuda")
    view = wide[:, 1:4, shift: shift + V]
    view.copy_(z)
    check(view, s, 6)
    turned = z.permute(1, 0, 2).contiguous().permute(1, 0, 2)  # beams outside
    check(turned, s, 6)
    check(z.transpose(1, 2).contiguous().transpose(1, 2), s, 6)  # tokens apart: copied


@pytest.mark.parametrize("V, n", [(9, 8), (3000, 16), (20000, 64), (70000, 64)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_ties_go_to_the_lower_beam_and_token(V, n, dtype):
    """All logits alike, and all beams: more equal candidates than any list holds."""
    z = torch.full((2, 8, V), 1.5, dtype=dtype, device="cuda")
    s = torch.full((2, 8), -3.0, device="cuda")
    got = check(z, s, n)
    assert got[1].tolist() == [[i // V for i in range(n)]] * 2 and got[2].tolist() == [[i % V for i in range(n)]] * 2
    z[:, :, ::3] = 2.0  # two values
    check(z, s, n)
    s[1] = torch.arange(8.0).neg() * 50
    check(z, s, n)


def test_values_in_few_threads():
    """A constrained vocabulary: -inf but for runs of tokens that few of a block's threads see."""
    z, s = spaced(1, 2, 3, 30000)
    keep = (torch.arange(30000, device="cuda") // 4) % 256 < 140
    z = torch.where(keep, z, -math.inf)
    check(z, s, 12)
    z = torch.where(torch.arange(30000, device="cuda") % 5000 == 17, z, -math.inf)  # six tokens
    check(z, s, 18)
    check(z, s, 40)  # fewer candidates than places


def test_the_types_lowest_value_is_a_logit():
    for dtype in (F32, BF):
        z, s = spaced(3, 1, 2, 500, dtype)
        z[:, :, 4:] = torch.finfo(dtype).min
        check(z, s, 8)
        z[:] = torch.finfo(dtype).min  # nothing else: all alike
        check(z, s, 8)
        z[:, :, 7] = torch.finfo(dtype).max
        check(z, s, 2)


# Wherever a row lies LSE holds, term by term: with d the mean distance of the row's terms from its maximum (at most log V,
# below 13 here) the exponents' rounding counts (d + 1) 2^-24, log2(e) in 32 bits d 2^-26, the exponential 2^-22 and sums of
# at most 16 values in 32 bits (two rounds, four sums a thread) 18 x 2^-24: together 2.4e-6, and LSE is 3.8e-6.
# The fills are of the kind that a constrained vocabulary is masked with, where -inf is not wanted.
FILLS = [-1e4, -1e6, -1e9, -1e10, -1e12, -1e16, -1e20, -1e30]


@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("V, shift", [(3000, 0), (20000, 0), (20001, 3)])
def test_a_vocabulary_masked_by_a_finite_value(fill, dtype, V, shift):
    """A handful of tokens is allowed, in pieces with none, a few and many of them; the rest is as good as absent."""
    from woodcock_b200.context import Context

    n = 6
    place = torch.arange(V, device="cuda")
    for allowed in (place % 1111 == 17, (place > 900) & (place < 900 + n), place < 300, place % 7 == 0, place == V - 5):
        want = n if allowed.sum() > 1 else 3
        for seed in range(20):
            z, s = spaced(seed, 2, 3, V, dtype)
            z = torch.where(allowed, z, fill).to(dtype)
            if selected(z, s, want)[3]:
                break
        wide = torch.full((2, 3, V + 8), math.nan, dtype=dtype, device="cuda")
        row = wide[:, :, shift: shift + V]
        row.copy_(z)
        got = check(row, s, want)
        assert allowed[got[2].long()].all()
    Context.get(0).synchronize()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_masked_values_in_several_rounds_of_a_piece(dtype):
    from woodcock_b200.context import Context

    place = torch.arange(65536, device="cuda")  # two rounds a piece
    allowed = torch.where(place % 16384 < 8192, place % 4096 == 5, place % 3 == 0)  # few in a round, many in the next
    for seed in range(8):
        z, s = spaced(seed, 64, 8, 65536, dtype)
        if selected(torch.where(allowed, z, -math.inf), s, 8)[3]:
            break
    for fill in (-1e10, -1e20):
        got = check(torch.where(allowed, z, fill).to(dtype), s, 8)
        assert allowed[got[2].long()].all()
    Context.get(0).synchronize()


@pytest.mark.parametrize("level", [1e10, -1e10, 1e16, -1e16, 1e20, -1e20, 1e30, -1e30, 2e38, -2e38])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_at_large_values_offer_their_tokens(level, dtype):
    """Whole rows, and single tokens above the others."""
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    z, s = spaced(43, 1, 2, 9000, dtype)
    assert (ops.beam_select(torch.full_like(z, level), s, 4)[0] > -math.inf).all()
    z[:, :, 4000] = level
    got = ops.beam_select(z, s, 1)
    assert (got[0] > -math.inf).all() and (got[2] == 4000).all() == (level > 0)
    Context.get(0).synchronize()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("levels", [(0, 20, -20), (0, 300, -300), (0, 1000, -1000), (1e4, 0, -1e5), (1e6, -1e6, 3e6), (-1e9, 1e9, 0),
                                    (1e12, -1e16, 2e38)])
def test_a_row_may_be_shifted(levels, dtype):
    """Beams at levels of their own, against the formula of what the type makes of them, with the bound that holds at 0.
    At the last levels a row is of one value and 64 bits hold lse in steps of 2^-13 and more, for both alike."""
    for V, n in ((700, 6), (20001, 9)):
        for seed in range(20):
            z, s = spaced(60 + seed, 2, 3, V)
            z = (z + torch.tensor(levels, device="cuda")[None, :, None]).to(dtype)
            if selected(z, s, n)[3]:
                break
        check(z, s, n, apart=False)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("fill", [-1e4, -1e6, -1e9, -1e10, -1e16, -1e20, -1e30, 1e9, 1e16, 2e38])
def test_rows_of_one_value(fill, dtype):
    """Every token has log-probability -log V, wherever the row lies (64 bits: log V in steps of 2^-53 of the level)."""
    s = torch.tensor([[-1.0, -2.0], [-7.0, -3.0]], device="cuda")
    for V in (50, 40000):
        z = torch.full((2, 2, V), fill, dtype=dtype, device="cuda")
        check(z, s, 7, apart=False)
        z[1, 0, V - 3] = 0.0 if fill < 0 else 3e38  # one token beside which the others are nothing
        check(z, s, 1, apart=False)


def test_dead_and_finished_beams():
    z, s = try_seeds(3, 6, 700, 12)
    first = torch.full_like(s, -math.inf)
    first[:, 0] = 0.0
    check(z, first, 6)  # a search begins
    check(z, torch.full_like(s, -math.inf), 6)  # nobody is left
    f = torch.zeros((3, 6), dtype=torch.bool, device="cuda")
    f[0, 2] = f[1, 0] = f[1, 5] = True
    f[2] = True
    z2 = z.clone()
    z2[0, 2] = math.nan  # an ended beam's logits may be anything
    z2[1, 5] = math.inf
    s[2, 3] = -math.inf
    z2[2, 3] = math.nan
    check(z2, s, 12, finished=f, pad=699)
    from woodcock_b200.context import Context

    Context.get(0).synchronize()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_no_number_raises_the_error_word(bad):
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    ctx.synchronize()
    z, s = spaced(5, 2, 3, 20000)
    z[0, 1, 19999] = bad
    check(z, s, 6, apart=False)
    with pytest.raises(WcError):
        ctx.synchronize()
    z[0, 1] = math.nan
    check(z, s, 6, apart=False)
    with pytest.raises(WcError):
        ctx.synchronize()
    z, s = spaced(5, 2, 3, 2000)
    s[1, 2] = bad
    check(z, s, 6, apart=False)
    with pytest.raises(WcError):
        ctx.synchronize()
    ctx.synchronize()


def test_arguments_of_select_that_are_refused():
    from woodcock_b200 import ops

    z, s = spaced(6, 2, 3, 50)
    f = torch.zeros((2, 3), dtype=torch.bool, device="cuda")
    for args, kw, what in (((z.double(), s), {}, "fp32 or bf16"), ((z, s.double()), {}, "scores"), ((z, s[:1]), {}, "scores"),
                           ((z, s.cpu()), {}, "scores"), ((z, s, 0), {}, "positive"), ((z, s, -1), {}, "positive"), ((z, s, 65), {}, "64"),
                           ((z, s), {"finished": f.int()}, "finished"), ((z, s), {"finished": f[:1]}, "finished"),
                           ((z, s), {"pad": 50}, "pad"), ((z, s), {"pad": -1}, "pad"), ((z[:, :, :0], s), {}, "token"),
                           ((z[:, :0], s[:, :0]), {}, "beam"), ((torch.zeros((1, 65, 9), device="cuda"), torch.zeros((1, 65), device="cuda")),
                                                                {}, "64 beams")):
        with pytest.raises(ValueError, match=what):
            ops.beam_select(*args, **kw)
    assert [x.shape for x in ops.beam_select(z[:0], s[:0])] == [(0, 3)] * 3


# ---------------------------------------------------------------------------- reordering


class Beams:
    def __init__(self, seed, lens, W, L, Hk, D, page, dtype, shared=0, cols=None):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.B, self.W, self.lens, self.page = len(lens), W, lens, page
        self.cols = cols or max(1, max(n // page + 1 for n in lens))
        tail = self.cols - shared
        total = self.B * (shared + W * tail) + 1
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        common = ids[: self.B * shared].view(self.B, 1, shared).expand(-1, W, -1)
        own = ids[self.B * shared: self.B * shared + self.B * W * tail].view(self.B, W, tail)
        self.table = torch.cat([common, own], 2).reshape(self.B * W, self.cols).contiguous()
        self.k, self.v = (torch.randn((L, total, Hk, page, D), generator=g, device="cuda").to(dtype) for _ in range(2))
        self.kv = i32([n for n in lens for _ in range(W)])

    def expect(self, parents):
        """The rule, beam by beam: the new table, k and v."""
        k, v, new = self.k.clone(), self.v.clone(), self.table.clone()
        for b, n in enumerate(self.lens):
            rows = [b * self.W + w for w in range(self.W)]
            p, full, rest = parents[b], n // self.page, n % self.page
            dead, taken = [w for w in range(self.W) if w not in p], set()
            for w in range(self.W):
                new[rows[w], :full] = self.table[rows[p[w]], :full]
                if rest:
                    heir = p[w] if p[w] not in taken else dead.pop(0)
                    new[rows[w], full] = self.table[rows[heir], full]
                    if p[w] in taken:
                        src, dst = int(self.table[rows[p[w]], full]), int(self.table[rows[heir], full])
                        k[:, dst, :, :rest] = self.k[:, src, :, :rest]
                        v[:, dst, :, :rest] = self.v[:, src, :, :rest]
                taken.add(p[w])
        return k, v, new

    def history(self, table, pool, row, n):
        at = torch.arange(n, device="cuda")
        return pool[:, table[row].long()[at // self.page], :, at % self.page]


def bits(x):
    return x.view(torch.int16 if x.element_size() == 2 else torch.int32)


def check_reorder(c, parents, **kw):
    from woodcock_b200 import ops

    k, v, new = c.expect(parents)
    before = [c.history(c.table, c.k, b * c.W + p, c.lens[b]).clone() for b, ps in enumerate(parents) for p in ps]
    got = ops.beam_reorder(c.k, c.v, c.table, c.kv, parents, **kw)
    assert torch.equal(got, new)
    assert torch.equal(bits(c.k), bits(k)) and torch.equal(bits(c.v), bits(v))
    for row, want in enumerate(before):  # what it is for: every beam has its parent's keys
        assert torch.equal(bits(c.history(got, c.k, row, c.lens[row // c.W])), bits(want))
    for b, n in enumerate(c.lens):  # and pages to fill of its own
        for col in range(n // c.page, c.cols):
            assert len(set(got[b * c.W: (b + 1) * c.W, col].tolist())) == c.W
    return got


@pytest.mark.parametrize("lens, W, L, Hk, D, page, dtype, shared, parents", [
    ([5], 1, 1, 1, 64, 16, BF, 0, [[0]]),
    ([33], 4, 3, 8, 128, 16, BF, 2, [[0, 0, 0, 0]]),
    ([33], 4, 3, 8, 128, 16, BF, 0, [[3, 2, 1, 0]]),
    ([40, 41], 4, 2, 2, 64, 16, F32, 1, [[1, 1, 3, 3], [2, 0, 2, 2]]),
    ([32, 64], 3, 2, 2, 64, 32, BF, 1, [[2, 2, 1], [0, 0, 0]]),   # full pages alone: nothing to copy
    ([0, 1], 3, 2, 2, 64, 16, BF, 0, [[2, 2, 1], [1, 1, 1]]),
    ([255], 5, 1, 3, 128, 256, F32, 0, [[4, 4, 4, 0, 0]]),
    ([19] * 7, 2, 2, 2, 128, 16, BF, 1, [[0, 1], [1, 0], [0, 0], [1, 1], [0, 1], [0, 0], [1, 1]]),
])
def test_reordering(lens, W, L, Hk, D, page, dtype, shared, parents):
    check_reorder(Beams(30, lens, W, L, Hk, D, page, dtype, shared), parents)


def test_64_beams_and_a_table_that_ends_with_the_keys():
    g = torch.Generator().manual_seed(3)
    c = Beams(31, [47, 64], 64, 2, 2, 64, 16, BF, cols=4)
    for _ in range(3):
        parents = torch.randint(0, 64, (2, 64), generator=g).tolist()
        c.table = check_reorder(c, parents)


def test_strided_pages_and_an_output_that_is_given():
    from woodcock_b200 import ops

    c = Beams(32, [23, 30], 3, 2, 4, 64, 16, BF)
    k, v, new = c.expect([[2, 2, 2], [1, 0, 0]])
    both = torch.zeros((c.k.shape[1], 2, 16, 4, 2, 64), dtype=BF, device="cuda")
    kk, vv = (both[:, :, :, :, i].permute(1, 0, 3, 2, 4) for i in range(2))
    kk.copy_(c.k), vv.copy_(c.v)
    wide = torch.full((6, 9), -5, dtype=torch.int32, device="cuda")
    wide[:, :2] = c.table
    out = torch.empty_like(c.table)
    assert ops.beam_reorder(kk, vv, wide[:, :2], c.kv, i32([[2, 2, 2], [1, 0, 0]]), out=out) is out
    assert torch.equal(out, new) and torch.equal(kk, k) and torch.equal(vv, v)


def test_pages_far_into_a_large_pool():
    """Offsets beyond 2^31 elements."""
    from woodcock_b200 import ops

    c = Beams(36, [23, 30], 3, 1, 8, 128, 16, BF)
    total, n = 140_000, c.k.shape[1]  # 16384 elements a page
    k, v = (torch.empty((total, 8, 16, 128), dtype=BF, device="cuda") for _ in range(2))
    k[total - n:], v[total - n:] = c.k[0], c.v[0]
    want = c.expect([[2, 2, 2], [1, 0, 0]])
    got = ops.beam_reorder(k, v, c.table + (total - n), c.kv, i32([[2, 2, 2], [1, 0, 0]]))
    assert torch.equal(got - (total - n), want[2])
    assert torch.equal(k[total - n:], want[0][0]) and torch.equal(v[total - n:], want[1][0])


def test_requests_that_are_left_as_they_are():
    from woodcock_b200 import ops
    from woodcock_b200._lib import WcError
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    ctx.synchronize()

    def spoil(c, what):
        table, kv, parents = c.table.clone(), c.kv.clone(), [[1, 1, 1], [0, 0, 2]]
        if what == "parent":
            parents[0][1] = 3
        elif what == "negative":
            parents[0][2] = -1
        elif what == "lengths":
            kv[1] = 22
        elif what == "long":
            kv[:3] = 33
        elif what == "below zero":
            kv[:3] = -1
        elif what == "page":
            table[2, 1] = c.k.shape[1]
        else:
            table[2, 1] = table[0, 1]
        return table, kv, parents

    for what in ("parent", "negative", "lengths", "long", "below zero", "page", "twice"):
        c = Beams(33, [23, 30], 3, 2, 2, 64, 16, BF)
        table, kv, parents = spoil(c, what)
        c.lens = [0, 30]  # of the first request nothing moves
        k, v, new = c.expect([[0, 1, 2], parents[1]])
        new[:3] = table[:3]
        got = ops.beam_reorder(c.k, c.v, table, kv, parents)
        with pytest.raises(WcError):
            ctx.synchronize()
        assert torch.equal(got, new) and torch.equal(c.k, k) and torch.equal(c.v, v), what
    ctx.synchronize()


def test_arguments_of_reorder_that_are_refused():
    from woodcock_b200 import ops

    c = Beams(34, [23, 30], 3, 2, 2, 64, 16, BF)
    p = i32([[0, 1, 2], [0, 1, 2]])
    for kw, what in (({"parents": p[:1]}, "parents"), ({"kv_lens": i32([1, 2])}, "entries"), ({"v_pages": c.k}, "share"),
                     ({"out": c.table}, "overlap"), ({"out": torch.empty((6, 3), dtype=torch.int32, device="cuda")}, "out must"),
                     ({"k_pages": c.k[0]}, "alike"), ({"out": c.k.view(torch.int32).view(-1)[:12].view(6, 2)}, "overlap"),
                     ({"kv_lens": c.v.view(torch.int32).view(-1)[:6]}, "overlap"),
                     ({"page_table": torch.zeros((65, 2), dtype=torch.int32, device="cuda"), "parents": i32([[0] * 65]), "kv_lens": i32([5] * 65)},
                      "64 beams")):
        args = {"k_pages": c.k, "v_pages": c.v, "page_table": c.table, "kv_lens": c.kv, "parents": p, **kw}
        with pytest.raises(ValueError, match=what):
            ops.beam_reorder(**args)


def test_captured_and_replayed_step():
    """Selection's parents go into the reordering on the device; the graph is replayed on other logits."""
    from woodcock_b200 import ops

    c = Beams(35, [23, 40], 4, 2, 2, 64, 16, BF)
    z, s = spaced(7, 2, 4, 9000)
    k0, v0 = c.k.clone(), c.v.clone()
    k, v = k0.clone(), v0.clone()

    def step(k, v):
        picked = ops.beam_select(z, s)
        return *picked, ops.beam_reorder(k, v, c.table, c.kv, picked[1])

    step(k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k, v)
    for seed in range(4):
        z2, s2 = spaced(50 + seed, 2, 4, 9000)
        z.copy_(z2), s.copy_(s2), k.copy_(k0), v.copy_(v0)
        graph.replay()
        c.k, c.v = k0.clone(), v0.clone()
        parents = selected(z, s, 4)[1].tolist()
        assert out[1].tolist() == parents
        want = c.expect(parents)
        assert torch.equal(out[3], want[2]) and torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_selections_on_streams_of_their_own():
    from woodcock_b200 import ops

    inputs = [try_seeds(2, 3 + i, 30000 + i, 8) for i in range(4)]
    want = [ops.beam_select(*x, 8) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, st in zip(inputs, streams):
            with torch.cuda.stream(st):
                got.append(ops.beam_select(*x, 8))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------------------- together


def test_a_beam_search_over_pages():
    """Beams over a prompt: append, attend, select, reorder, step after step, against every beam's own dense
    history. The 'model' reads the attention's output through a fixed head."""
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    B, W, H, Hk, D, page, V, prompt, steps = 2, 4, 4, 2, 64, 16, 600, 21, 24
    g = torch.Generator(device="cuda").manual_seed(40)
    R = lambda *n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    emb, head = R(V, (H + 2 * Hk) * D), R(H * D, V) * 0.8
    cols = (prompt + steps) // page + 1
    shared = prompt // page
    total = B * (shared + W * (cols - shared))
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.cat([ids[: B * shared].view(B, 1, shared).expand(-1, W, -1),
                       ids[B * shared:].view(B, W, cols - shared)], 2).reshape(B * W, cols).contiguous()
    k, v = (torch.full((total, Hk, page, D), math.nan, device="cuda") for _ in range(2))

    def rows(tokens):
        x = emb[tokens].view(-1, H + 2 * Hk, D)
        return x[:, :H], x[:, H: H + Hk], x[:, H + Hk:]

    # the prompt goes into beam 0's pages; then every beam continues beam 0
    tokens = torch.randint(0, V, (B * prompt,), generator=g, device="cuda")
    q, kn, vn = rows(tokens)
    first = table.view(B, W, cols)[:, 0].contiguous()
    qr = ops.paged_append(q, kn, vn, k, v, first, i32([prompt] * B))
    out = ops.paged_attention(qr, k, v, first, i32([prompt] * B))
    table = ops.beam_reorder(k, v, table, i32([prompt] * (B * W)), torch.zeros((B, W), dtype=torch.int32))
    last = out.view(B, prompt, H * D)[:, -1:].expand(B, W, H * D)
    scores = torch.full((B, W), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    # every beam's history of rotated keys and values: the plain side
    rot = ops.paged_append(kn.contiguous(), kn, vn, torch.zeros_like(k), torch.zeros_like(v), first, i32([prompt] * B))
    hist = [[(rot[b * prompt: (b + 1) * prompt], vn[b * prompt: (b + 1) * prompt])] * W for b in range(B)]
    forks = 0
    for step in range(steps):
        logits = (last @ head).contiguous()
        want = selected(logits, scores, W)
        scores, parents, picked = ops.beam_select(logits, scores)
        if want[3]:
            assert torch.equal(parents.cpu().long(), want[1]) and torch.equal(picked.cpu().long(), want[2])
        n = prompt + step
        table = ops.beam_reorder(k, v, table, i32([n] * (B * W)), parents)
        par = parents.tolist()
        forks += sum(W - len(set(p)) for p in par)
        hist = [[hist[b][p] for p in par[b]] for b in range(B)]
        q, kn, vn = rows(picked.view(-1).long())
        kv = i32([n + 1] * (B * W))
        qr = ops.paged_append(q, kn, vn, k, v, table, kv)
        out = ops.paged_attention(qr, k, v, table, kv)
        kr = ops.paged_append(kn.contiguous(), kn, vn, torch.zeros_like(k), torch.zeros_like(v), table, kv)
        for b in range(B):
            for w in range(W):
                i = b * W + w
                K, X = (torch.cat([x, y[i: i + 1]]) for x, y in zip(hist[b][w], (kr, vn)))
                hist[b][w] = (K, X)
                K, X = (x.double().repeat_interleave(H // Hk, 1) for x in (K, X))
                p = torch.softmax(torch.einsum("hd,khd->hk", qr[i].double(), K) * D ** -0.5, -1)
                o = torch.einsum("hk,khd->hd", p, X)
                a = torch.einsum("hk,khd->hd", p, X.abs())
                # the 32-bit attention's bound: scores off by (head_dim + 4) 2^-24 sum |q k| scale < 2^-11 here
                assert ((out[i].double() - o).abs() <= 2.0 ** -9 * a).all(), (step, b, w)
        last = out.view(B, W, H * D)
    assert forks > 10
    Context.get(0).synchronize()
