"""head_logprobs on the GPU in every form that its sizes choose: few and many loads of a ring, pairs of blocks with long sums, large vocabularies."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from test_gpu_head_logprobs import check, some

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
