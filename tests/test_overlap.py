"""The checks of overlapping memory (csrc/overlap.h) against sets of bytes, without a GPU."""

from __future__ import annotations

import subprocess

from conftest import REPO


def test_overlaps_are_those_of_the_bytes(tmp_path):
    exe = tmp_path / "overlap"
    subprocess.run(["g++", "-std=c++17", "-O1", str(REPO / "tests" / "overlap.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
