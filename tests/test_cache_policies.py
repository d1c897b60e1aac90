"""What the eviction and beam search operators refuse, and their argument layout, without a GPU."""

from __future__ import annotations

import subprocess

import pytest
import torch

from conftest import REPO


def _pages(dtype=torch.bfloat16, dim=64, size=16):
    return torch.zeros((3, 2, size, dim), dtype=dtype)


TABLE, LENS = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)


@pytest.mark.parametrize("k, what", [
    (_pages(torch.float16), "fp32 or bf16"),
    (_pages()[0], "pages must be"),
    (_pages().transpose(2, 3), "contiguous"),
    (_pages(dim=96), "head_dim"),
    (_pages(size=24), "page_size"),
    (_pages(), "CUDA"),
])
def test_pages_that_are_refused(k, what):
    from woodcock_b200 import ops

    mass, q = torch.zeros(k.shape[:-1]), torch.zeros((1, 4, 64), dtype=k.dtype)
    with pytest.raises(ValueError, match=what):
        ops.paged_mass(q, k, mass, TABLE, LENS)
    with pytest.raises(ValueError, match=what):
        ops.paged_evict(k, k.clone(), mass, TABLE, LENS, 4)
    with pytest.raises(ValueError, match=what):
        ops.beam_reorder(k, k.clone(), TABLE, LENS, [[0]])


@pytest.mark.parametrize("logits, what", [
    (torch.zeros((2, 3, 10), dtype=torch.float16), "fp32 or bf16"),
    (torch.zeros((6, 10)), "requests"),
    (torch.zeros((2, 3, 10)), "CUDA"),
])
def test_logits_that_are_refused(logits, what):
    from woodcock_b200 import ops

    with pytest.raises(ValueError, match=what):
        ops.beam_select(logits, torch.zeros((2, 3)))


def test_null_handles_are_refused():
    from woodcock_b200._lib import WC_ERR_INVALID, lib

    L = lib()
    for call in (L.wc_paged_mass, L.wc_paged_mass_workspace, L.wc_paged_evict, L.wc_paged_evict_workspace, L.wc_beam_select,
                 L.wc_beam_select_workspace, L.wc_beam_reorder):
        assert call(None, None, None) == WC_ERR_INVALID


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    from woodcock_b200 import beam, paged

    # every struct, and where the header has some of its fields: each is found again after packing
    fields = {"wc_paged_mass_args": (paged._MASS, ["q", "mass", "workspace", "scale", "layer", "add"]),
              "wc_paged_evict_args": (paged._EVICT, ["mass", "page_table", "requests", "lens_out", "workspace_bytes", "recent"]),
              "wc_beam_select_args": (beam._SELECT, ["beam_stride", "finished", "out_tokens", "workspace", "dtype", "pad"]),
              "wc_beam_reorder_args": (beam._REORDER, ["page_table", "beams", "kv_lens", "parents", "table_out", "out_stride"])}
    src = tmp_path / "sizes.c"
    src.write_text('#include "woodcock_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) {\n' + "".join(
        f'  printf("%zu", sizeof({t}));\n' + "".join(f'  printf(" %zu", offsetof({t}, {f}));\n' for f in names) +
        '  printf("\\n");\n' for t, (_, names) in fields.items()) + "  return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    index = {"wc_paged_mass_args": [24, 27, 31, 33, 34, 35], "wc_paged_evict_args": [16, 20, 23, 26, 28, 31],
             "wc_beam_select_args": [2, 4, 7, 8, 10, 15], "wc_beam_reorder_args": [16, 20, 22, 23, 24, 25]}
    for line, (name, (fmt, _)) in zip(lines, fields.items()):
        size, *offsets = map(int, line.split())
        assert size == fmt.size, name
        for i, at in zip(index[name], offsets):
            values = [0.0 if isinstance(v, float) else 0 for v in fmt.unpack(bytes(size))]
            zeros = fmt.pack(*values)
            values[i] = 1.0 if isinstance(values[i], float) else 1
            changed = [j for j, (x, y) in enumerate(zip(zeros, fmt.pack(*values))) if x != y]
            assert at <= changed[0] < at + 4, (name, i)
