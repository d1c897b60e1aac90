"""Threads that share a context: each is told its own failure, none of the shared words is raced on."""

from __future__ import annotations

import subprocess
import threading
import time

from conftest import REPO


def test_failures_and_launches_of_threads(tmp_path):
    cmd = ["g++", "-std=c++17", "-O1", "-I", "/usr/local/cuda/include", "-I", str(REPO / "include"),
           str(REPO / "tests" / "host_threads.cpp"), "-o", str(tmp_path / "t")]
    flags = ["-fsanitize=thread"]
    (tmp_path / "e.cpp").write_text("int main() { return 0; }\n")
    if subprocess.run(["g++", *flags, str(tmp_path / "e.cpp"), "-o", str(tmp_path / "e")], capture_output=True).returncode \
            or subprocess.run([str(tmp_path / "e")], capture_output=True).returncode:
        flags = []  # no sanitizer: the messages and counts are still compared
    subprocess.run([*cmd, *flags], check=True, capture_output=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ThreadSanitizer" not in r.stderr, r.stdout + r.stderr[:2000]


def test_threads_that_ask_first_get_one_context(monkeypatch):
    from woodcock_b200.context import Context

    made, got, start = [], [], threading.Barrier(8)

    def init(self, device=0):
        time.sleep(0.05)
        made.append(device)

    def ask():
        start.wait()
        got.append(Context.get(5))

    monkeypatch.setattr(Context, "__init__", init)
    monkeypatch.setattr(Context, "_by_device", {})
    threads = [threading.Thread(target=ask) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert made == [5] and len({id(c) for c in got}) == 1


def test_a_paged_call_makes_its_context_within_the_device(monkeypatch):
    """Making a context selects its device; the one that was current comes back."""
    import torch

    from woodcock_b200 import paged
    from woodcock_b200.context import Context

    current = [0]

    class device:
        def __init__(self, d):
            self.d = d.index

        def __enter__(self):
            self.before, current[0] = current[0], self.d

        def __exit__(self, *_):
            current[0] = self.before

    def init(self, index=0):
        current[0] = index  # as the library does

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(Context, "__init__", init)
    monkeypatch.setattr(Context, "_by_device", {})
    a = paged._context(torch.device("cuda", 3))
    assert current == [0] and paged._context(torch.device("cuda", 3)) is a and Context.get(3) is a
