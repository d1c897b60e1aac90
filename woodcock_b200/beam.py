"""Beam search over the paged cache (wc_beam_* in the C ABI): which continuations survive, and their pages.

The reference keeps one continuation per request (python/woodcock/spec.py:151-212). Here a request has several
beams, each with a page table, a length and a row of logits of its own; to the paged operators every beam is a
request. One step: append and attend over all beams, project to logits, ``beam_select``, then
``beam_reorder``, whose table the next step takes. Work runs on the caller's current stream, scratch comes from
PyTorch's allocator for the one call; scores, parents, tables and lengths stay on the device, so a captured
graph can be replayed on new contents.
"""

from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache

import torch

from ._lib import lib
from .paged import _CODES, _PAGES, _context, _fail, _ints, _pages, _stream, _table

# wc_beam_select_args and wc_beam_reorder_args of the header, in their native layout
_SELECT = struct.Struct("@P2q6PQ6i0q")
_REORDER = struct.Struct("@" + _PAGES + "Pq4i3Pq0q")


@lru_cache(maxsize=4096)
def _select_workspace(device: int, code: int, requests: int, beams: int, vocab: int, n: int) -> int:
    size = C.c_uint64()
    ctx = _context(torch.device("cuda", device))
    ctx.check(lib().wc_beam_select_workspace(ctx.h, _SELECT.pack(
        16, 0, 0, 16, 0, 16, 16, 16, 0, 0, code, requests, beams, vocab, n, 0), C.byref(size)))
    return size.value


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int | None = None, finished: torch.Tensor | None = None,
                pad: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The n best continuations of each request over its beams and the vocabulary, best first:
    (scores fp32, parents int32, tokens int32), each [requests][n].

    logits [requests][beams][vocab] fp32 or bf16, any strides with contiguous tokens; scores fp32
    [requests][beams], the beams' log probabilities so far (-inf: a dead beam, as all but the first are at the
    start). A continuation's score is scores[w] + log_softmax(logits[w])[token]; ties go to the lower beam, then
    to the lower token. Ranks are decided in 64 bits, the scores given are rounded to 32; the exponentials behind a
    beam's log_softmax are of 32 bits, which leaves its scores within 2^-18 of the formula's wherever the row lies (calls of
    up to 70 million logits; beyond, at worst in proportion). n: default the number of beams, at most 64
    (twice the beams leaves enough where some end); at most 64 beams.

    ``finished`` (bool [requests][beams]): a beam that has ended offers itself alone, with its score and token
    ``pad``; its logits are not looked at, nor a dead beam's. A token at -inf is never chosen; places for which no
    candidate is left hold -inf, parent 0, token 0. A beam whose logits or score hold NaN or +inf offers nothing and
    raises the context's device error word."""
    if logits.dim() != 3 or logits.dtype not in _CODES:
        _fail("logits must be [requests][beams][vocab], fp32 or bf16")
    dev, (B, W, V) = logits.device, logits.shape
    if not logits.is_cuda:
        _fail("logits must be on a CUDA device")
    if scores.dtype is not torch.float32 or scores.shape != (B, W) or scores.device != dev:
        _fail("scores must be fp32 [requests][beams] on the logits' device")
    if finished is not None and (finished.dtype is not torch.bool or finished.shape != (B, W) or finished.device != dev):
        _fail("finished must be bool [requests][beams] on the logits' device")
    n = W if n is None else n
    if V == 0 or W == 0:
        _fail("beam_select needs a beam and a token")
    ls = logits.stride()
    if V > 1 and ls[2] != 1 or ls[0] < 0 or ls[1] < 0:
        logits = logits.contiguous()
        ls = logits.stride()
    scores = scores.contiguous()
    finished = None if finished is None else finished.contiguous()
    if n <= 0:
        _fail("n must be positive")
    out, parents, tokens = scores.new_empty((B, n)), *scores.new_empty((2, B, n), dtype=torch.int32).unbind()
    if B == 0:
        return out, parents, tokens
    ctx = _context(dev)
    device = ctx.device.index
    code = _CODES[logits.dtype]
    size = _select_workspace(device, code, B, W, V, n)
    ws = scores.new_empty(size + 256, dtype=torch.uint8)
    ctx.check(lib().wc_beam_select(ctx.h, _stream(device), _SELECT.pack(
        logits.data_ptr(), ls[0], ls[1], scores.data_ptr(), 0 if finished is None else finished.data_ptr(), out.data_ptr(),
        parents.data_ptr(), tokens.data_ptr(), -(-ws.data_ptr() // 256) * 256, size, code, B, W, V, n, pad)))
    return out, parents, tokens


def beam_reorder(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table, kv_lens, parents,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Gives every beam its parent's keys, in every layer; returns the beams' new page table (int32
    [requests * beams][pages of a beam]).

    Pages [layers][pages][kv_heads][page_size][head_dim] or one layer's; page_table [requests * beams][cols];
    kv_lens int32 [requests * beams], alike for the beams of a request (they stay as they are); parents int32
    [requests][beams], the beam of the request that each beam continues from now on.

    A page that is full is shared: the new table names the parent's. The page that is being filled has to be another
    one for each beam, as have those behind it: a parent's first child (the lowest beam) keeps it, the i-th further
    child of the request takes the page of the i-th beam that has no child, and the filled rows are copied there.
    So a request needs one page per beam and column, whatever happens, and at most one page per beam is copied. To
    start a search, fill beam 0's pages with the prompt, give all beams its length and use parents 0 throughout.

    A request with a parent out of range, beams of unequal length, a length beyond the table, or a page being filled
    that lies outside the pool or in two beams' tables is left as it is and raises the device error word. At most 64
    beams. ``out`` must not overlap page_table."""
    dev = k_pages.device
    pages = _pages(k_pages, v_pages, layers=k_pages.dim() == 5)
    table = _table(page_table, dev, "page_table")
    rows, cols = table.shape
    parents = _table(parents, dev, "parents").contiguous()
    B, W = parents.shape
    if B * W != rows:
        _fail("parents must be [requests][beams], page_table a row for each")
    lens = _ints(kv_lens, dev, rows, "kv_lens")
    if out is None:
        out = table.new_empty((rows, cols))
    elif out.shape != (rows, cols) or out.dtype is not torch.int32 or out.device != dev or not out.is_contiguous():
        _fail(f"out must be a contiguous ({rows}, {cols}) int32 tensor on {dev}")
    if rows == 0:
        return out
    ctx = _context(dev)
    ctx.check(lib().wc_beam_reorder(ctx.h, _stream(ctx.device.index), _REORDER.pack(
        *pages, table.data_ptr(), table.stride(0) if rows > 1 else cols, cols, B, W, 0, lens.data_ptr(),
        parents.data_ptr(), out.data_ptr(), cols)))
    return out
