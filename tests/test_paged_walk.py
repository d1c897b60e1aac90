"""The blocks' walk over the line of key tiles (PagedWalk in paged.cuh) on CPU threads, under the thread
sanitizer: no block's shared memory is accessed without a barrier between, whether it has work or not,
and the blocks' shares are the line, each tile once."""

from __future__ import annotations

import random
import subprocess

import pytest

from conftest import REPO

CUDA_INCLUDE = "/usr/local/cuda/include"
M, KT, OVER = 128, 128, 3  # as instantiated in paged_walk.cpp


def build(out, *flags):
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=thread", *flags, "-I", CUDA_INCLUDE, "-I", str(REPO / "include"),
                    str(REPO / "tests" / "paged_walk.cpp"), "-o", str(out)], check=True, capture_output=True)


@pytest.fixture(scope="module")
def sanitizer(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "t.cpp").write_text("int main() { return 0; }\n")
    if subprocess.run(["g++", "-fsanitize=thread", str(d / "t.cpp"), "-o", str(d / "t")], capture_output=True).returncode \
            or subprocess.run([str(d / "t")], capture_output=True).returncode:
        pytest.skip("no thread sanitizer")
    return d


def text(cases):
    out = [str(len(cases))]
    for c in cases:
        out.append(" ".join(str(c[k]) for k in ("B", "G", "H", "Hk", "page_log2", "tree", "grid", "least", "kinds")))
        out += [" ".join(map(str, c[k])) for k in ("lens", "offsets", "plens", "groups")]
    return "\n".join(out) + "\n"


def case(lens, rows, H, Hk, grid, least, plens=(), groups=(), kinds=1, tree=0, page_log2=4):
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    return {"B": len(lens), "G": len(plens), "H": H, "Hk": Hk, "page_log2": page_log2, "tree": tree, "grid": grid,
            "least": least, "kinds": kinds, "lens": lens, "offsets": off, "plens": list(plens), "groups": list(groups)}


def line(c):
    """The items in order: (prefix, index, head, row tile, key tiles)."""
    segs, rep = [], c["H"] // c["Hk"]
    if c["kinds"] & 2:
        for g in range(c["G"]):
            segs.append((1, g, c["offsets"][c["groups"][g + 1]] - c["offsets"][c["groups"][g]], c["plens"][g]))
    if c["kinds"] & 1:
        segs += [(0, b, c["offsets"][b + 1] - c["offsets"][b], c["lens"][b]) for b in range(c["B"])]
    items = []
    for prefix, i, n, klen in segs:
        for head in range(c["Hk"]):
            for qt in range(-(-n * rep // M)):
                seen = klen
                if not prefix and not c["tree"]:
                    seen = min(max(klen - n + min(n - 1, ((qt + 1) * M - 1) // rep) + 1, 0), klen)
                items.append((prefix, i, head, qt, max(1, -(-seen // KT))))
    return items


def shares(c):
    """Each block's (item, first tile, last, tiles, first block, blocks)."""
    items = line(c)
    total = sum(x[4] + OVER for x in items)
    per = max(c["least"], -(-total // c["grid"]))
    out, at = [[] for _ in range(c["grid"])], 0
    for x in items:
        a = at + OVER  # the item's first tile; the units before it hold none
        first, last = a // per, (a + x[4] - 1) // per
        for b in range(first, last + 1):
            lo, hi = max(a, b * per), min(a + x[4], (b + 1) * per)
            out[b].append((*x[:4], lo - a, hi - a, x[4], first, last - first + 1))
        at += x[4] + OVER
    return out


def drawn(rng):
    B = rng.choice([1, 2, 5, 40, 500])
    Hk = rng.choice([1, 2, 8])
    rows = [rng.choice([0, 1, 2, 30, 130, 300]) for _ in range(B)]
    lens = [rng.choice([0, 1, r, r + 127, r + 128, rng.randrange(4000)]) for r in rows]
    G = rng.choice([0, 0, 1, min(3, B)])
    cuts = sorted(rng.randrange(B + 1) for _ in range(G + 1)) if G else []
    kinds = rng.choice([1, 2, 3]) if G else 1
    return case(lens, rows, Hk * rng.choice([1, 2, 5]), Hk, rng.choice([1, 3, 8]), rng.choice([1, 4]),
                [rng.randrange(3000) for _ in range(G)], cuts, kinds, rng.choice([0, 1]) if max(rows) <= 64 else 0)


# few units for many blocks: most have no work
IDLE = [case([40], [10], 1, 1, 8, 4), case([70, 60], [20, 20], 8, 2, 8, 4, [500], [0, 2], 2, 1),
        case([0], [0], 2, 1, 8, 1), case([3] * 3, [1, 0, 2], 4, 1, 8, 4)]


def test_blocks_share_the_line_without_a_race(sanitizer):
    rng = random.Random(7)
    cases = IDLE + [drawn(rng) for _ in range(12)]
    exe = sanitizer / "walk"
    build(exe)
    for _ in range(3):
        r = subprocess.run([str(exe)], input=text(cases), capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and "ThreadSanitizer" not in r.stderr, r.stderr[:2000]
    got = []
    for row in r.stdout.splitlines():
        w = row.split()
        if w[0] == "case":
            got.append([])
        elif w[0] == "block":
            assert w[2] == "1"  # the second walk from the kept beginning is the first one
            got[-1].append([])
        else:
            got[-1][-1].append(tuple(map(int, w)))
    assert len(got) == len(cases)
    for c, blocks in zip(cases, got):
        assert blocks == shares(c), c
    assert any(not b for b in got[0])


def test_a_walk_kept_by_every_block_is_reported(sanitizer):
    """Thread 0 of a block without work stores over words that other warps still sum: the sanitizer (or the
    walk itself, with the total that it then reads) ends the run."""
    exe = sanitizer / "always"
    build(exe, "-DSTORE_ALWAYS")
    for _ in range(5):
        try:
            r = subprocess.run([str(exe)], input=text(IDLE * 4), capture_output=True, text=True, timeout=60)
        except subprocess.TimeoutExpired:  # or meets a barrier alone
            return
        if r.returncode != 0:
            return
    pytest.fail("not reported")
