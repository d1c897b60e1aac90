"""Calls of the paged operators that their documentation allows beyond those of test_gpu_paged.py, and
refusals of those that it does not. Tolerances: test_gpu_paged.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF, Case, check, i32

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
