"""The paged operators' refusals and argument layout, without a GPU."""

from __future__ import annotations

import subprocess

import pytest
import torch

from conftest import REPO


def _pages(pages=3, heads=2, size=16, dim=64, dtype=torch.bfloat16):
    return torch.zeros((pages, heads, size, dim), dtype=dtype)


@pytest.mark.parametrize("k, v, what", [
    (_pages(dtype=torch.float16), _pages(dtype=torch.float16), "fp32 or bf16"),
    (_pages(), _pages(dtype=torch.float32), "alike"),
    (_pages(), _pages(pages=4), "alike"),
    (_pages()[0], _pages()[0], "pages must be"),
    (_pages().transpose(2, 3), _pages().transpose(2, 3), "contiguous"),
    (_pages(dim=96), _pages(dim=96), "head_dim"),
    (_pages(size=24), _pages(size=24), "page_size"),
    (_pages(size=8), _pages(size=8), "page_size"),
    (_pages(), _pages(), "CUDA"),
])
def test_pages_that_are_refused(k, v, what):
    from woodcock_b200 import ops

    q = torch.zeros((1, 4, 64), dtype=k.dtype)
    table, lens = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match=what):
        ops.paged_attention(q, k, v, table, lens)
    with pytest.raises(ValueError, match=what):
        ops.paged_append(q, q, q, k, v, table, lens)
    with pytest.raises(ValueError, match=what):
        ops.shared_prefix_attention(q, k, v, table, lens, [0, 1], table, lens)
    if k.dim() == 4:  # a 3-D pool is no pool for compaction either, but says so in other words
        with pytest.raises(ValueError, match=what):
            ops.paged_compact(k, v, table, lens, table, lens)


def test_null_handles_are_refused():
    from woodcock_b200._lib import WC_ERR_INVALID, lib

    L = lib()
    assert L.wc_paged_append(None, None, None) == WC_ERR_INVALID
    assert L.wc_paged_attention(None, None, None) == WC_ERR_INVALID
    assert L.wc_paged_attention_workspace(None, None, None) == WC_ERR_INVALID
    assert L.wc_paged_compact(None, None, None) == WC_ERR_INVALID


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    from woodcock_b200 import paged

    src = tmp_path / "sizes.c"
    src.write_text('#include "woodcock_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) {\n'
                   '  printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(wc_paged_append_args), '
                   'sizeof(wc_paged_attention_args), sizeof(wc_paged_compact_args), '
                   'offsetof(wc_paged_append_args, layer), offsetof(wc_paged_attention_args, layer), '
                   'offsetof(wc_paged_compact_args, max_keep));\n  return 0;\n}\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes[:3] == [paged._APPEND.size, paged._ATTENTION.size, paged._COMPACT.size]
    # the last integer field lands where the header has it
    for fmt, n, at in ((paged._APPEND, sizes[0], sizes[3]), (paged._ATTENTION, sizes[1], sizes[4]),
                       (paged._COMPACT, sizes[2], sizes[5])):
        values = list(fmt.unpack(bytes(n)))
        values[-1] = 0x01020304
        assert fmt.pack(*values)[at : at + 4] == bytes([4, 3, 2, 1])
