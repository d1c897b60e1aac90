"""Operators over a paged KV cache, for batches of requests of unequal length (wc_paged_* in the C ABI).

The reference decodes one request over one contiguous cache (include/woodcock/cache.h:9-28,
python/woodcock/target.py:159-175); a server keeps many requests' keys and values in pages instead.

* Pages: ``k_pages`` and ``v_pages`` are [pages][kv_heads][page_size][head_dim], fp32 or bf16, any
  strides that are multiples of 16 bytes with contiguous rows. head_dim is 64 or 128, page_size a
  power of two from 16 to 256. Key j of request b is row j % page_size of page
  ``page_table[b][j // page_size]`` (int32).
* ``kv_lens`` (int32 [requests]) counts each request's keys, its new rows included: append and
  attention take the same lengths. Request b's new rows are rows q_offsets[b] .. q_offsets[b + 1] of
  q, k, v and out (int32 [requests + 1]; None: rows / requests each); rows behind the last request
  are left alone.
* Tables, lengths and offsets stay on the device, so a captured CUDA graph can be replayed on new
  contents (make one call before the capture). A page number outside the pool (its keys and values read
  as zeros), a length beyond its table (cut to it) or a row with no slot (its k and v are dropped) is never
  followed; it raises the context's device error word (``Context.get(device).synchronize()`` after
  the stream's work raises WcError).
* ``mass_pages`` (fp32 [pages][kv_heads][page_size]) hold the attention weight that each key has gathered, beside
  the pages and addressed by the same tables; rows contiguous, any other strides.
* Work runs on the caller's current stream of the tensors' device, in its order; scratch comes from
  PyTorch's allocator for that one call. What a call writes (its output, the pages of append,
  compact and evict, the mass) must not overlap what it reads, nor itself: refused with ValueError. K and V may be cut from
  one buffer (halves, or side by side in a page, a head or a row). Several threads may call these
  operators at once, each with buffers of its own.
"""

from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache
from numbers import Integral

import torch

from ._lib import WC_BF16, WC_F32, lib
from .context import Context, device_ints

_CODES = {torch.float32: WC_F32, torch.bfloat16: WC_BF16}

# wc_pages, wc_paged_batch and the argument structs of the header, in their native layout
_PAGES = "2P8q6i"
_BATCH = "Pq2i2P2i"
_APPEND = struct.Struct("@" + _PAGES + _BATCH + "3P6q4Pdf2i0q")
_ATTENTION = struct.Struct("@" + _PAGES + _BATCH + "P2qPPq2P2i2PQfi0q")
_COMPACT = struct.Struct("@" + _PAGES + "Pq2i2Pq2Pi0q")
_MASS = struct.Struct("@" + _PAGES + _BATCH + "P2qP3qPQf2i0q")
_EVICT = struct.Struct("@" + _PAGES + "P3qPq2i4PQ3i0q")

_raw_stream = torch._C._cuda_getCurrentRawStream


def _fail(what: str):
    raise ValueError(what)


def _context(device: torch.device) -> Context:
    ctx = Context._by_device.get(device.index)
    if ctx is None:  # making one selects its device: the caller's stays the current one
        with torch.cuda.device(device):
            ctx = Context.get(device)
    return ctx


def _stream(device: int) -> int:
    # the default stream's handle is 0, which the library reads as "the context's"; 1 names it
    return _raw_stream(device) or 1


def _pages(k: torch.Tensor, v: torch.Tensor, layers: bool = False) -> tuple:
    code, n = _CODES.get(k.dtype), k.shape
    if code is None or v.dtype is not k.dtype:
        _fail("pages must be fp32 or bf16, k and v alike")
    if len(n) != 4 + layers or v.shape != n:
        _fail(f"pages must be {'[layers]' if layers else ''}[pages][kv_heads][page_size][head_dim], k and v alike")
    ks, vs = k.stride(), v.stride()
    if ks[-1] != 1 or vs[-1] != 1:
        _fail("rows of the pages must be contiguous")
    if n[-1] not in (64, 128) or n[-2] not in (16, 32, 64, 128, 256):
        _fail("head_dim must be 64 or 128, page_size a power of two from 16 to 256")
    if not k.is_cuda or v.device != k.device:
        _fail("pages must be on one CUDA device")
    if layers:
        return (k.data_ptr(), v.data_ptr(), *ks[:4], *vs[:4], code, n[1], n[3], n[2], n[4], n[0])
    return (k.data_ptr(), v.data_ptr(), 0, ks[0], ks[1], ks[2], 0, vs[0], vs[1], vs[2], code, n[0], n[2], n[1], n[3], 1)


def _ints(x, device, n: int, name: str) -> torch.Tensor:
    if not (isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.device == device and x.dim() == 1
            and x.is_contiguous()):
        x = device_ints(x, device)
    if x.shape[0] != n:
        _fail(f"{name} must have {n} entries")
    return x


def _table(x, device, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x)
    if x.dim() != 2:
        _fail(f"{name} must be [requests][pages of a request]")
    if x.dtype is not torch.int32 or x.device != device:
        x = x.to(device=device, dtype=torch.int32)
    if not x.is_contiguous():
        n, st = x.shape, x.stride()
        if n[1] and st[1] != 1 or n[0] > 1 and st[0] < n[1]:
            x = x.contiguous()
    return x


def _rows(x: torch.Tensor, dtype, device, heads: int | None, head_dim: int, rows: int | None, name: str) -> tuple:
    """(the tensor whose memory is read, its first two strides, its shape)"""
    n = x.shape
    if len(n) != 3 or n[2] != head_dim or (heads is not None and n[1] != heads) or (rows is not None and n[0] != rows):
        _fail(f"{name} must be [rows][heads][head_dim] to match the pages and q")
    if x.dtype is not dtype or x.device != device:
        _fail(f"{name} must be {dtype} on {device}")
    s, unit = x.stride(), 8 if dtype is torch.bfloat16 else 4
    if s[2] != 1 or s[0] % unit or s[1] % unit or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s = x.stride()
    return x, s, n


def _batch(T: int, H: int, table, kv_lens, q_offsets, device) -> tuple:
    table = _table(table, device, "page_table")
    B, cols = table.shape
    lens = _ints(kv_lens, device, B, "kv_lens")
    off = None if q_offsets is None else _ints(q_offsets, device, B + 1, "q_offsets")
    if off is None and (T % B if B else T):
        _fail("without q_offsets, q's rows must be a multiple of the requests")
    # the tensors come back too: a converted one must live until the launch
    return (table.data_ptr(), table.stride(0) if B > 1 else cols, cols, B, lens.data_ptr(),
            0 if off is None else off.data_ptr(), T, H), B, (table, lens, off)


def _out(out, x: torch.Tensor, shape, dtype) -> torch.Tensor:
    if out is None:
        return x.new_empty(shape, dtype=dtype)
    if out.shape != shape or out.dtype is not dtype or out.device != x.device or not out.is_contiguous():
        _fail(f"out must be a contiguous {tuple(shape)} {dtype} tensor on {x.device}")
    return out


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table, kv_lens, positions=None, q_offsets=None, base: float = 1e6,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Normalises, rotates and appends new rows; returns the rotated q in the pages' dtype.

    q [rows][heads][head_dim], k and v [rows][kv_heads][head_dim], fp32 or bf16 (views of a fused
    projection's output are read in place). With gains q_norm / k_norm ([head_dim]) each head is
    RMS-normalised first (ops.rmsnorm, eps). q and k are rotated as ops.rope does, at ``positions``
    (int32 [rows]; None: the row's place among its request's keys) with angles in 64 bits, so that any
    position up to 2^31 keeps its angle. The new rows become the last of kv_lens[b] keys. Two rows of
    one call must not fall on the same page slot."""
    dev = k_pages.device
    pages = _pages(k_pages, v_pages)
    D, Hk, src = pages[14], pages[13], q.dtype
    if src not in _CODES:
        _fail("q must be fp32 or bf16")
    q, qs, shape = _rows(q, src, dev, None, D, None, "q")
    T = shape[0]
    k, ks, _ = _rows(k, src, dev, Hk, D, T, "k")
    v, vs, _ = _rows(v, src, dev, Hk, D, T, "v")
    batch, B, keep = _batch(T, shape[1], page_table, kv_lens, q_offsets, dev)
    pos = None if positions is None else _ints(positions, dev, T, "positions")
    gains = []
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None:
            if w.shape != (D,):
                _fail(f"{name} must be [head_dim]")
            if w.dtype is not torch.float32 or w.device != dev or not w.is_contiguous() or w.data_ptr() % 16:
                w = w.to(device=dev, dtype=torch.float32, copy=True).contiguous()
        gains.append(w)
    qn, kn = gains
    out = _out(out, q, shape, k_pages.dtype)
    if T == 0 or B == 0:
        return out
    ctx = _context(dev)
    ctx.check(lib().wc_paged_append(ctx.h, _stream(ctx.device.index), _APPEND.pack(
        *pages, *batch, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
        0 if pos is None else pos.data_ptr(), 0 if qn is None else qn.data_ptr(), 0 if kn is None else kn.data_ptr(),
        out.data_ptr(), base, eps, _CODES[src], 0)))
    return out


@lru_cache(maxsize=4096)
def _workspace(device: int, code: int, pages: int, page_size: int, kv_heads: int, head_dim: int, cols: int,
               requests: int, rows: int, heads: int, groups: int) -> int:
    """Bytes of scratch for calls of these sizes (the library looks at no buffer for this)."""
    n = C.c_uint64()
    ctx = _context(torch.device("cuda", device))
    st = head_dim * page_size * kv_heads
    strides = (0, st, head_dim * page_size, head_dim)
    ctx.check(lib().wc_paged_attention_workspace(ctx.h, _ATTENTION.pack(
        16, 16, *strides, *strides, code, pages, page_size, kv_heads, head_dim, 1, 16, cols, cols, requests, 16, 16,
        rows, heads, 16, 0, 0, 0, 16, 0, 16, 16, groups, 0, 16, 0, 0, 1.0, 0), C.byref(n)))
    return n.value


def _attend(q, k_pages, v_pages, prefix, page_table, kv_lens, q_offsets, tree_mask, scale, out):
    dev = k_pages.device
    pages = _pages(k_pages, v_pages)
    D, kind = pages[14], k_pages.dtype
    q, qs, shape = _rows(q, kind, dev, None, D, None, "q")
    T, H, _ = shape
    batch, B, keep = _batch(T, H, page_table, kv_lens, q_offsets, dev)
    if tree_mask is not None:
        if tree_mask.dtype is not torch.int64 or tree_mask.shape != (T,) or tree_mask.device != dev:
            _fail("tree_mask must be int64 [rows], a bit for each of the request's new rows")
        tree_mask = tree_mask.contiguous()
    G, pre = 0, (0, 0, 0, 0, 0, 0)
    if prefix is not None:
        table = _table(prefix[0], dev, "prefix_table")
        G, cols = table.shape
        plens, ends = _ints(prefix[1], dev, G, "prefix_lens"), _ints(prefix[2], dev, G + 1, "group_offsets")
        pre = (table.data_ptr(), table.stride(0) if G > 1 else cols, plens.data_ptr(), ends.data_ptr(), G, cols)
    out = _out(out, q, shape, kind)
    if T == 0 or B == 0:
        return out
    ctx = _context(dev)
    device = ctx.device.index
    n = _workspace(device, pages[10], pages[11], pages[12], pages[13], D, batch[2], B, T, H, G)
    ws = q.new_empty(n + 256, dtype=torch.uint8)
    ctx.check(lib().wc_paged_attention(ctx.h, _stream(device), _ATTENTION.pack(
        *pages, *batch, q.data_ptr(), qs[0], qs[1], 0 if tree_mask is None else tree_mask.data_ptr(), *pre,
        out.data_ptr(), -(-ws.data_ptr() // 256) * 256, n, D ** -0.5 if scale is None else scale, 0)))
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table, kv_lens,
                    q_offsets=None, tree_mask: torch.Tensor | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged batch over its pages: softmax(scale q K^T) V per head, [rows][heads][head_dim].

    q [rows][heads][head_dim] of the pages' dtype, heads a multiple of kv_heads; decoding steps,
    verification chains, draft trees and prompts may share a call. New row i of a request sees the keys
    before the new rows and new rows 0..i; with ``tree_mask`` (int64 [rows], at most 64 new rows a
    request) those new rows whose bit is set. A row that sees nothing gives 0; masked places may hold
    anything, NaN and infinities included. Statistics and sums are fp32; with bf16 pages the softmax
    weights are rounded to bf16 once (at most 2^-8 of each; ops.attention, which takes and returns fp32,
    keeps two bf16 terms). scale: positive, default head_dim ** -0.5.

    The kernel follows from rows / requests over the whole call, so where a few prompts have most of the
    rows and steps most of the requests, one call for each kind is faster than one for both."""
    return _attend(q, k_pages, v_pages, None, page_table, kv_lens, q_offsets, tree_mask, scale, out)


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, prefix_table, prefix_lens,
                            group_offsets, page_table, kv_lens, q_offsets=None, tree_mask: torch.Tensor | None = None,
                            scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention for requests that share prefixes: each prefix is read once for all of its rows.

    Group g is requests group_offsets[g] .. group_offsets[g + 1] (int32 [groups + 1]; requests outside
    every group have no prefix); its rows all see the prefix_lens[g] keys in pages prefix_table[g],
    besides what paged_attention shows them of page_table / kv_lens, which hold only the request's own
    keys. The prefix's and the own part's softmax states are joined in fp32, one rounding at the end."""
    return _attend(q, k_pages, v_pages, (prefix_table, prefix_lens, group_offsets), page_table, kv_lens, q_offsets,
                   tree_mask, scale, out)


def paged_compact(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table, starts, keep, n_keep) -> torch.Tensor:
    """Moves accepted rows together after a verification (KVCache.compact over pages, all requests and
    layers): key starts[b] + keep[b][i] -> starts[b] + i for i < n_keep[b]; returns the new lengths
    starts + n_keep (int32).

    Pages [layers][pages][kv_heads][page_size][head_dim] or one layer's; keep int32
    [requests][at most 64], strictly increasing. A request with a bad list keeps its rows and raises the
    device error word. Requests must not share the pages that their moved rows lie in."""
    dev = k_pages.device
    pages = _pages(k_pages, v_pages, layers=k_pages.dim() == 5)
    table = _table(page_table, dev, "page_table")
    B, cols = table.shape
    starts = _ints(starts, dev, B, "starts")
    n_keep = _ints(n_keep, dev, B, "n_keep")
    keep = _table(keep, dev, "keep")
    most = keep.shape[1]
    if keep.shape[0] != B or most < 1:
        _fail("keep must be [requests][at least 1]")
    lens = starts.new_empty(B)
    if B == 0:
        return lens
    ctx = _context(dev)
    many = B > 1
    ctx.check(lib().wc_paged_compact(ctx.h, _stream(ctx.device.index), _COMPACT.pack(
        *pages, table.data_ptr(), table.stride(0) if many else cols, cols, B, starts.data_ptr(), keep.data_ptr(),
        keep.stride(0) if many else most, n_keep.data_ptr(), lens.data_ptr(), most)))
    return lens


def _mass(mass: torch.Tensor, pages: torch.Tensor) -> tuple:
    n = pages.shape[:-1]
    if mass.dtype is not torch.float32 or mass.shape != n or mass.device != pages.device:
        _fail(f"mass_pages must be fp32 {list(n)} on {pages.device}: the pages without head_dim")
    s = mass.stride()
    if s[-1] != 1:
        _fail("rows of mass_pages must be contiguous")
    return (mass.data_ptr(), *s[:3]) if len(n) == 4 else (mass.data_ptr(), 0, *s[:2])


@lru_cache(maxsize=4096)
def _mass_workspace(device: int, code: int, pages: int, page_size: int, kv_heads: int, head_dim: int, cols: int,
                    requests: int, ragged: int, rows: int, heads: int) -> int:
    n = C.c_uint64()
    ctx = _context(torch.device("cuda", device))
    st = head_dim * page_size * kv_heads
    strides = (0, st, head_dim * page_size, head_dim)
    ctx.check(lib().wc_paged_mass_workspace(ctx.h, _MASS.pack(
        16, 16, *strides, *strides, code, pages, page_size, kv_heads, head_dim, 1, 16, cols, cols, requests, 16, 16 * ragged,
        rows, heads, 16, 0, 0, 16, 0, 0, 0, 0, 0, 1.0, 0, 0), C.byref(n)))
    return n.value


def paged_mass(q: torch.Tensor, k_pages: torch.Tensor, mass_pages: torch.Tensor, page_table, kv_lens, q_offsets=None,
               scale: float | None = None, add: bool = True) -> torch.Tensor:
    """Adds up the attention weight that each key gathers, for paged_evict; returns mass_pages.

    mass[b][kv head][key] = was + the sum over request b's new rows and the kv head's query heads of
    softmax(scale q K^T)[key], the weights that paged_attention gives without a tree_mask. q as there
    ([rows][heads][head_dim] of the pages' dtype). ``was`` is what the key gathered before: 0 for the keys that
    are new in this call (a page may hold anything before), and with ``add=False`` for all of them, so that the
    keys of a request without rows have 0 then. Rows need not be all that were appended: after a verification the
    accepted ones, behind a prompt its last ones. A row that sees nothing adds nothing. Statistics and sums are
    fp32, in the same order every time. Beside what the additions of its score and of the sums round, a weight is
    within 2^-20 + 2^-22 |s| of itself, s the row's score of largest magnitude times log2(e): with bf16 pages and more
    than 16 rows a head the row's maximum and the logarithm of its sum are held as one fp32 number.

    Requests must not share pages, since two would write a sum: with a common prompt each needs keys of its own. A
    call whose requests have more pages than the pool because they do raises the device error word, and the pages'
    sums are not to be used; sharing of fewer pages goes unnoticed."""
    dev = k_pages.device
    pages = _pages(k_pages, k_pages)
    D, kind = pages[14], k_pages.dtype
    mass = _mass(mass_pages, k_pages)
    q, qs, shape = _rows(q, kind, dev, None, D, None, "q")
    T, H, _ = shape
    batch, B, keep = _batch(T, H, page_table, kv_lens, q_offsets, dev)
    if B == 0:
        return mass_pages
    ctx = _context(dev)
    device = ctx.device.index
    n = _mass_workspace(device, pages[10], pages[11], pages[12], pages[13], D, batch[2], B,
                        q_offsets is not None, T, H) if T else 0
    ws = q.new_empty(n + 256, dtype=torch.uint8)
    ctx.check(lib().wc_paged_mass(ctx.h, _stream(device), _MASS.pack(
        *pages, *batch, q.data_ptr(), qs[0], qs[1], *mass, -(-ws.data_ptr() // 256) * 256, n,
        D ** -0.5 if scale is None else scale, 0, bool(add))))
    return mass_pages


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, mass_pages: torch.Tensor, page_table, kv_lens, budget,
                sinks: int = 0, recent: int = 0) -> torch.Tensor:
    """Brings every request within its budget of keys; returns the new lengths min(kv_lens, budget) (int32).

    Each layer and kv head of a request with more keys keeps ``budget`` of them (an int, or int32 [requests]): the
    first ``sinks``, the last ``recent``, and of those between the ones of the largest mass (ties: the lower key;
    a NaN ranks last). They become keys 0 .. budget - 1 in their order, with their mass; what lies behind is left as
    it was. Keys keep the rotation they were appended with, so later rows need explicit positions.

    Pages [layers][pages][kv_heads][page_size][head_dim] with mass [layers][pages][kv_heads][page_size], or one
    layer's. A request whose budget is below sinks + recent keeps everything and raises the device error word.
    Requests must not share pages. Scratch is 4 bytes for each layer, request, kv head and key of the budget; with
    budgets on the device, of the table's width in keys, so that tables no wider than needed save memory."""
    dev = k_pages.device
    pages = _pages(k_pages, v_pages, layers=k_pages.dim() == 5)
    mass = _mass(mass_pages, k_pages)
    table = _table(page_table, dev, "page_table")
    B, cols = table.shape
    lens = _ints(kv_lens, dev, B, "kv_lens")
    most, budgets = cols * pages[12], None
    if isinstance(budget, Integral):
        budget = int(budget)
        if budget < sinks + recent:
            _fail("budget must not be below sinks + recent")
        budget = min(budget, 0x7FFFFFFF)
        most = min(most, budget)
    else:
        budgets, budget = _ints(budget, dev, B, "budget"), 0
    if not 0 <= sinks < 1 << 30 or not 0 <= recent < 1 << 30:
        _fail("sinks and recent must not be negative")
    out = lens.new_empty(B)
    if B == 0:
        return out
    ctx = _context(dev)
    n = pages[15] * B * pages[13] * (most + 1) * 4
    ws = k_pages.new_empty(n + 256, dtype=torch.uint8)
    ctx.check(lib().wc_paged_evict(ctx.h, _stream(ctx.device.index), _EVICT.pack(
        *pages, *mass, table.data_ptr(), table.stride(0) if B > 1 else cols, cols, B, lens.data_ptr(),
        0 if budgets is None else budgets.data_ptr(), out.data_ptr(), -(-ws.data_ptr() // 256) * 256, n, budget, sinks,
        recent)))
    return out
