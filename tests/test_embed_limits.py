"""The lookup's gradient at the largest vocabulary and the longest list of
tokens: the kernels' counts stay inside int (constant evaluation refuses an
overflow), and the sums are right there."""
import os
import subprocess

import pytest
import torch

from gene2vec_amd import build as B
from gene2vec_amd import ops

TOP = 2**31 - 1


def test_counts_do_not_overflow():
    def up(n, size):
        return -(-n // size)
    checks = []
    for n in (0, 1, 255, 256, 257, TOP - 256, TOP - 255, TOP - 1, TOP):
        for size in (1, 256, 4096, 2**21 - 1, 2**21, TOP):
            checks.append((f"pieces({n}, {size})", up(n, size)))
        for log2 in (0, 6, 8):
            checks.append((f"pieces_log2({n}, {log2})", up(n, 1 << log2)))
    for V in (1, 255, 256, 257, TOP - 255, TOP):
        for b in (0, 1, 254, 255):
            checks.append((f"rows_of_bucket({V}, {b}, 256)", len(range(b, V, 256))))
    source = '#include "g2v_counts.h"\n' + "".join(
        f'static_assert(g2v::{call} == {want}, "");\n' for call, want in checks)
    r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-x", "c++", "-I", B.CSRC, "-"],
                       input=source, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]


def test_kernels_use_the_checked_counts():
    """no rounded-up division by an addition is left on the device side"""
    src = open(os.path.join(B.CSRC, "g2v_embed.hip")).read()
    device = src[:src.index("struct Plan")]
    for line in ("rows_of_bucket(V, b, kBuckets)", "pieces(n, hot)", "pieces_log2(run.y, s.log2L)"):
        assert line in device
    for line in ("+ kBuckets - 1", "n + hot - 1", "run.y + "):
        assert line not in device


@pytest.mark.gpu
def test_gradient_of_the_largest_vocabulary():
    ids = [TOP - 1, 3, TOP - 256, 3, 255, -1, 2**30 + 7]
    dy = torch.arange(1.0, len(ids) + 1, device="cuda")[:, None].to(torch.bfloat16)
    g = ops.embedding_lookup_grad(dy, torch.tensor(ids, device="cuda"), TOP)
    for row, want in ((TOP - 1, 1), (3, 6), (TOP - 256, 3), (255, 5), (2**30 + 7, 7)):
        assert float(g[row]) == want
        g[row] = 0
    assert not any(bool(part.any()) for part in g.split(2**28))


@pytest.mark.gpu
def test_gradient_of_the_longest_list():
    """2^31 - 1 tokens, nearly all of one row: its bucket is cut into parts and
    its run into pieces.  Whole numbers of few bits: exact in any order"""
    ids = torch.full((TOP,), 5, dtype=torch.int32, device="cuda")
    ids[7], ids[TOP - 9], ids[TOP - 8] = 261, 4, 900
    dy = torch.zeros(TOP, 1, dtype=torch.bfloat16, device="cuda")
    for at, v in ((0, 1), (7, 8), (2**30, 2), (TOP - 9, 16), (TOP - 8, 32), (TOP - 1, 64)):
        dy[at] = v
    g = ops.embedding_lookup_grad(dy, ids, 300).float().cpu().flatten()
    want = torch.zeros(300)
    want[5], want[261], want[4] = 1 + 2 + 64, 8, 16
    assert torch.equal(g, want)
