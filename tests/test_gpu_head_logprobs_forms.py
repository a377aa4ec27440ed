"""head_logprobs on the GPU in every form that its sizes choose: few and many loads of a ring, pairs of blocks with long sums, large vocabularies."""
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
