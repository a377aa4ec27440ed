"""head_logprobs on the GPU in every form that its sizes choose: few and many loads of a ring, pairs of blocks with long sums, large vocabularies."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from test_gpu_head_logprobs import check, some

from nano_vllm_b200 import _lib
from nano_vllm_b200.logprobs import head_logprobs
from oracle.logprobs_ref import assert_same, head_logprobs_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,stages", [(4, 11), (128, 6), (200, 6)])
def test_loads_around_the_stages_of_the_ring(cuda, rows, stages):
    """One block and a pair of them with fewer loads than stages, as many, and a few more: the last stages' ends are waited for."""
    g = torch.Generator().manual_seed(rows)
    for blocks in (1, 2, stages - 1, stages, stages + 1, 2 * stages, 2 * stages + 1):
        check(cuda, *some(g, rows, 64 * blocks, 190))


def test_forms_that_only_a_graph_has(cuda):
    """A process whose first eager call is of one row captures a call of every other form."""
    script = """
import sys
sys.path[:0] = ["tests", "."]
import torch
from test_gpu_head_logprobs import some
from nano_vllm_b200.logprobs import head_logprobs
g = torch.Generator().manual_seed(1)
cases = [[t.cuda() for t in some(g, rows, hidden, 700)] for rows, hidden in ((1, 64), (140, 64), (1, 1536), (140, 1536))]
head_logprobs(*cases[0])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = [head_logprobs(*c) for c in cases]
graph.replay()
assert all(torch.equal(i, j) for o, c in zip(out, cases) for i, j in zip(o, head_logprobs(*c)))
"""
    done = subprocess.run([sys.executable, "-c", script], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("rows,hidden,vocab", [(600, 1536, 30011), (300, 2056, 9001), (1500, 1032, 5003), (2000, 4096, 300), (769, 1040, 2000)])
def test_pairs_with_long_sums(cuda, rows, hidden, vocab):
    """Parts of more than 1024 elements by pairs of blocks, whose row tiles divide the multiprocessors (300 rows) and do not."""
    g = torch.Generator().manual_seed(rows)
    check(cuda, *some(g, rows, hidden, vocab))


def test_long_sums_in_groups_of_tiles(cuda):
    """So many rows that a unit of work has several column tiles; rows from everywhere against the reference."""
    g = torch.Generator().manual_seed(9)
    x, w, tokens = some(g, 20_000, 1040, 20_011)
    got = head_logprobs(x.to(cuda), w.to(cuda), tokens.to(cuda))
    rows = torch.cat([torch.arange(3), torch.randint(20_000, (60,), generator=g), torch.arange(19_990, 20_000)])
    given, entropy, bounds = head_logprobs_ref(x[rows], w, tokens[rows])
    assert_same(got.logprobs[rows.to(cuda)], given, bounds[0], "logprobs")
    assert_same(got.entropy[rows.to(cuda)], entropy, bounds[1], "entropy")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("rows,hidden", [(3, 64), (140, 8), (2, 1032)])
def test_large_vocabularies(cuda, rows, hidden):
    """The largest there is, and a ragged one: the last columns' tokens are scored too."""
    g = torch.Generator().manual_seed(hidden)
    for vocab in ((1 << 21, 151_643) if hidden < 1000 else (151_643,)):
        x, w, tokens = some(g, rows, hidden, vocab)
        tokens[0], tokens[1] = vocab - 1, 0
        check(cuda, x, w, tokens)
