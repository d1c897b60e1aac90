"""Calls of the paged operators that their documentation allows beyond those of test_gpu_paged.py, and
refusals of those that it does not. Tolerances: test_gpu_paged.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF, F32, Case, check, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H, Hk, rows, lens, prefix", [
    (2, 1, 20, [40, 21], [130]),       # a few blocks of work for the whole device, on the 128-row kernel
    (16, 8, 10, [70], [64, 0]),
    (4, 1, 300, [300, 301], [500]),    # the 256-row kernel
])
def test_blocks_without_work_leave_the_others_alone(H, Hk, rows, lens, prefix):
    from woodcock_b200 import ops
    from woodcock_b200.context import Context

    B = len(lens)
    c = Case(60, lens, [rows] * B, H, Hk, 128, 16, BF, prefix=prefix)
    groups = [min(g, B) for g in range(len(prefix) + 1)]
    call = lambda: (ops.paged_attention(c.q, c.k, c.v, c.table, c.kv),  # noqa: E731
                    ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, i32(prefix), i32(groups), c.table, c.kv))
    own, joined = call()
    check(c, own)
    check(c, joined, groups=groups)
    for _ in range(300):
        a, b = call()
        assert torch.equal(a, own) and torch.equal(b, joined)
    Context.get(0).synchronize()


def test_threads_that_are_refused_at_once_are_told_their_own_reasons():
    import threading

    from woodcock_b200 import ops

    c = Case(61, [40, 50], [1, 1], 16, 8, 128, 16, BF)
    n = c.q[:, :8].contiguous()
    keep = torch.zeros((2, 65), dtype=torch.int32, device="cuda")
    calls = {"scale": lambda: ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, scale=-1.0),
             "share": lambda: ops.paged_append(c.q, n, n, c.k, c.k, c.table, c.kv),
             "64": lambda: ops.paged_compact(c.k, c.v, c.table, c.kv, keep, i32([0, 0]))}
    told = {what: [] for what in calls}

    def run(what):
        for _ in range(300):
            try:
                calls[what]()
            except ValueError as e:
                told[what].append(str(e))

    threads = [threading.Thread(target=run, args=(what,)) for what in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for what, words in told.items():
        assert len(words) == 300 and all(what in w for w in words), (what, set(words))


def windows(x, step):
    """The pool with its pages `step` elements apart, each reaching into the next."""
    return x.as_strided(x.shape, (step, *x.stride()[1:]))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_written_memory_that_overlaps_is_refused(dtype):
    from woodcock_b200 import ops

    c = Case(62, [40, 50], [1, 1], 16, 8, 128, 16, dtype)
    n = torch.randn((2, 8, 128), generator=c.g, device="cuda").to(dtype)
    page = c.k[0].numel()
    zeros = i32([0, 0])

    def append(k, v, q=c.q, kn=n, vn=n, **kw):
        return ops.paged_append(q, kn, vn, k, v, c.table, c.kv, **kw)

    def compact(k, v, keep=None):
        return ops.paged_compact(k, v, c.table, zeros, i32([[0], [0]]) if keep is None else keep, zeros)

    both = torch.zeros((2 * c.k.shape[0], *c.k.shape[1:]), dtype=dtype, device="cuda")
    half = c.k.shape[0]
    for k, v, what in (
            (windows(c.k, page // 2), c.v, "overlap"),                # pages that reach into the next
            (c.k, windows(c.v, page - 128), "overlap"),
            (both[:half], both[1: half + 1], "share"),                # K and V a page apart in one buffer
            (both[: half], both[half - 1: 2 * half - 1], "share"),
            (both.view(half, 2, 8, 16, 128)[:, 0], both.view(half, 2, 8, 16, 128)[:, 0], "share")):
        for call in (append, compact):
            with pytest.raises(ValueError, match=what):
                call(k, v)
    flat = torch.zeros(2 * half * page + 2 * 16 * 128, dtype=dtype, device="cuda")
    pools = flat[: 2 * half * page].view(2, half, 8, 16, 128)
    k, v = pools[0], pools[1]
    inside = flat[2 * half * page - 2048: 2 * half * page + 2048].view(2, 16, 128)  # its first half in V's last page
    with pytest.raises(ValueError, match="overlap"):
        append(k, v, out=inside)
    with pytest.raises(ValueError, match="overlap"):
        append(k, v, q=inside)
    for kn, vn in ((k[0, :, :2].transpose(0, 1), n), (n, v[3, :, 4:6].transpose(0, 1))):
        with pytest.raises(ValueError, match="overlap"):
            append(k, v, kn=kn, vn=vn)
    with pytest.raises(ValueError, match="overlap"):
        ops.paged_attention(c.q, k, v, c.table, c.kv, out=inside)
    with pytest.raises(ValueError, match="overlap"):  # page numbers inside the pages
        ops.paged_compact(k, v, k.view(torch.int32)[0, 0, :2, : c.table.shape[1]], zeros, i32([[0], [0]]), zeros)
    # what lies apart is not refused: behind the pages, and K and V side by side in one buffer
    out = flat[2 * half * page:].view(2, 16, 128)
    assert append(k, v, out=out) is out
    assert ops.paged_attention(c.q, k, v, c.table, c.kv, out=out) is out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["halves", "page", "head", "row", "shifted"])
def test_k_and_v_in_one_buffer(dtype, layout):
    """Pools cut from one buffer: halves of it, or K and V of a page, a head or a row side by side."""
    from woodcock_b200 import ops

    c = Case(63, [40, 5, 90], [2, 2, 2], 8, 4, 64, 16, dtype)
    P, Hk, page, D = c.k.shape
    shape = {"halves": (2, P, Hk, page, D), "page": (P, 2, Hk, page, D), "head": (P, Hk, 2, page, D),
             "row": (P, Hk, page, 2, D), "shifted": (P + 4, 2, Hk, page, D)}[layout]
    buf = torch.full(shape, 3.0, dtype=dtype, device="cuda")
    axis = {"halves": 0, "page": 1, "head": 2, "row": 3, "shifted": 1}[layout]
    k, v = buf.select(axis, 0), buf.select(axis, 1)
    if layout == "shifted":
        k, v = k[:P], v[4:]
    k.copy_(c.k)
    v.copy_(c.v)
    new = [c.randn(6, h, D) for h in (8, 4, 4)]
    a = ops.paged_append(*new, c.k, c.v, c.table, c.kv)
    b = ops.paged_append(*new, k, v, c.table, c.kv)
    assert torch.equal(a, b)
    c.q = a
    out = ops.paged_attention(a, k, v, c.table, c.kv)
    check(c, out)
    assert torch.equal(out, ops.paged_attention(a, c.k, c.v, c.table, c.kv))
    args = c.table, i32([38, 3, 88]), i32([[0, 1], [1, 0], [1, 0]]), i32([2, 1, 1])
    assert torch.equal(ops.paged_compact(k, v, *args), ops.paged_compact(c.k, c.v, *args))
    assert torch.equal(k.nan_to_num(7.0), c.k.nan_to_num(7.0)) and torch.equal(v.nan_to_num(7.0), c.v.nan_to_num(7.0))


def test_a_workspace_over_what_the_call_reads_or_writes_is_refused():
    import ctypes as C

    from woodcock_b200 import ops, paged
    from woodcock_b200._lib import WC_ERR_INVALID, WC_OK, lib
    from woodcock_b200.context import Context

    ctx = Context.get(0)
    c = Case(64, [40, 50], [1, 1], 16, 8, 128, 16, BF)
    pages = paged._pages(c.k, c.v)
    batch, _, _ = paged._batch(2, 16, c.table, c.kv, None, c.k.device)
    need = C.c_uint64()
    out = torch.zeros((2, 16, 128), dtype=BF, device="cuda")

    def args(ws, n, to=out):
        return paged._ATTENTION.pack(*pages, *batch, c.q.data_ptr(), *c.q.stride()[:2], 0, 0, 0, 0, 0, 0, 0, to.data_ptr(), ws, n,
                                     128 ** -0.5, 0)

    assert lib().wc_paged_attention_workspace(ctx.h, args(16, 0), C.byref(need)) == WC_OK
    n = need.value
    buf = torch.zeros(2 * n + 512, dtype=torch.uint8, device="cuda")
    ws = -(-buf.data_ptr() // 256) * 256
    stream = paged._stream(0)
    for to in (ws, ws + n - 256):
        over = buf[to - buf.data_ptr():][: out.numel() * 2].view(BF).view(out.shape)
        assert lib().wc_paged_attention(ctx.h, stream, args(ws, n, over)) == WC_ERR_INVALID
    for x in (c.q, c.k, c.v):
        assert lib().wc_paged_attention(ctx.h, stream, args(-(-x.data_ptr() // 256) * 256, n)) == WC_ERR_INVALID
    over = buf[ws + n - buf.data_ptr():][: out.numel() * 2].view(BF).view(out.shape)  # right behind it
    assert lib().wc_paged_attention(ctx.h, stream, args(ws, n, over)) == WC_OK
    assert torch.equal(over, ops.paged_attention(c.q, c.k, c.v, c.table, c.kv))


FIRST_USE = """
import sys
sys.path[:0] = [{tests!r}, {repo!r}]
import torch
from test_gpu_paged import BF, F32, Case, check, i32
from woodcock_b200 import ops

c = Case(70, [40], [1], 16, 8, 128, 16, BF)
ops.paged_attention(c.q, c.k, c.v, c.table, c.kv)
torch.cuda.synchronize()
for c in (Case(71, [300, 200], [130, 20], 16, 8, 128, 16, BF, prefix=[100]), Case(72, [300], [300], 16, 8, 64, 16, BF, prefix=[100]),
          Case(73, [90, 80], [3, 3], 4, 2, 64, 16, F32, prefix=[100]), Case(74, [90, 80], [20, 3], 4, 2, 64, 16, BF, prefix=[100])):
    B, new = len(c.lens), [c.randn(sum(c.rows), h, c.D) for h in (c.H, c.Hk, c.Hk)]
    k, v, plens, ends = c.k.clone(), c.v.clone(), i32([100]), i32([0, B])
    starts, keep, n = i32([0] * B), i32([[0, 2]] * B), i32([2] * B)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        own = ops.paged_attention(c.q, c.k, c.v, c.table, c.kv, q_offsets=c.off)
        joined = ops.shared_prefix_attention(c.q, c.k, c.v, c.ptable, plens, ends, c.table, c.kv, q_offsets=c.off)
        q = ops.paged_append(*new, k, v, c.table, c.kv, q_offsets=c.off)
        lens = ops.paged_compact(k, v, c.table, starts, keep, n)
    g.replay()
    torch.cuda.synchronize()
    check(c, own)
    check(c, joined, groups=[0, B])
    k2, v2 = c.k.clone(), c.v.clone()
    assert torch.equal(q, ops.paged_append(*new, k2, v2, c.table, c.kv, q_offsets=c.off))
    assert torch.equal(lens, ops.paged_compact(k2, v2, c.table, starts, keep, n))
    assert torch.equal(k.nan_to_num(7.0), k2.nan_to_num(7.0)) and torch.equal(v.nan_to_num(7.0), v2.nan_to_num(7.0))
print("captured")
"""


def test_a_capture_may_hold_sizes_that_no_call_had_before():
    """One call of any size comes before a capture; the captured calls reach other kernels for the first time."""
    import subprocess
    import sys

    from conftest import REPO

    r = subprocess.run([sys.executable, "-c", FIRST_USE.format(tests=str(REPO / "tests"), repo=str(REPO))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_a_padded_batch_in_a_step():
    """Rows that pad a batch behind the last request hold NaN and are left alone by every operator of the step."""
    from woodcock_b200 import ops

    c = Case(65, [40, 5, 90], [2, 1, 3], 16, 8, 128, 16, BF)
    T, pad = 6, 5
    full = [torch.full((T + pad, h, 128), float("nan"), dtype=BF, device="cuda") for h in (16, 8, 8)]
    new = [c.randn(T, h, 128) for h in (16, 8, 8)]
    for x, y in zip(full, new):
        x[:T] = y
    k, v, out = c.k.clone(), c.v.clone(), torch.full((T + pad, 16, 128), 5.0, dtype=BF, device="cuda")
    a = ops.paged_append(*new, c.k, c.v, c.table, c.kv, q_offsets=c.off)
    assert ops.paged_append(*full, k, v, c.table, c.kv, q_offsets=c.off, out=out) is out
    assert torch.equal(out[:T], a) and (out[T:] == 5).all()
    assert torch.equal(k.nan_to_num(7.0), c.k.nan_to_num(7.0)) and torch.equal(v.nan_to_num(7.0), c.v.nan_to_num(7.0))
    c.q = a
    full[0][:T] = a
    got = ops.paged_attention(full[0], c.k, c.v, c.table, c.kv, q_offsets=c.off, out=torch.full_like(out, 5.0))
    check(c, got)
    assert (got[T:] == 5).all()
