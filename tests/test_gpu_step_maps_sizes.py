"""step_maps at sizes where a launch's resources change."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from nano_vllm_b200 import _lib, attention as A
from nano_vllm_b200.step_maps import step_maps

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

# In a process of its own: what the first launch on a device sets up must do for every later one, and for this one.
SCRIPT = r"""
import sys
sys.path[:0] = [%(root)r, %(root)r + "/tests"]
import torch
from nano_vllm_b200 import _lib
from oracle import fp8_cache_ref as F8
from nano_vllm_b200.step_maps import step_maps
batch = %(batch)d
g = torch.Generator().manual_seed(batch)
cached = torch.randint(0, 700, (batch,), generator=g, dtype=torch.int32)
seq = cached + torch.randint(0, 20, (batch,), generator=g, dtype=torch.int32)
table = torch.randint(-1, 50, (batch, 3), generator=g, dtype=torch.int32)
free, rows = torch.arange(batch, dtype=torch.int32) + 9000, int((seq - cached).sum()) + 3
dev = [t.cuda() for t in (seq, cached, table, free)]
m = step_maps(*dev, rows)
want = F8.step_maps_ref(seq, cached, table, free, rows)
assert dev[2].tolist() == want[0] and [t.tolist() for t in m[:4]] == [list(x) for x in want[1:5]] and m.blocks_taken.tolist() == [want[5]]
assert _lib.read_status() == 0
print("as listed")
"""


@pytest.mark.parametrize("batch", [3060, 3066, 3068, 3071, 4096])
def test_first_batch_of_a_process(cuda, batch):
    """16 bytes a sequence reach the 48 KB that a launch has without asking for more, beside what the kernel has of its own."""
    r = subprocess.run([sys.executable, "-c", SCRIPT % {"root": str(ROOT), "batch": batch}], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as listed" in r.stdout, r.stderr[-2000:]


def test_more_tokens_than_rows_stay_within_the_rows(cuda):
    """Offsets end at the rows there are: a prefill over them leaves what lies behind its output as it was."""
    i32 = dict(dtype=torch.int32, device=cuda)
    hq, hkv, d, rows = 4, 2, 64, 100
    codes, scales = torch.zeros(8, 256, hkv, d, device=cuda).to(torch.float8_e4m3fn), torch.ones(8, hkv, 16, device=cuda)
    q = torch.randn(rows, hq, d, device=cuda).bfloat16()
    for lens, want in (([300, 500], [0, 100, 100]), ([60, 500], [0, 60, 100]), ([60, 40], [0, 60, 100])):
        table = torch.full((2, 2), -1, **i32)
        _lib.read_status()
        m = step_maps(torch.tensor(lens, **i32), torch.zeros(2, **i32), table, torch.arange(8, **i32), rows)
        assert _lib.read_status() == (1 if sum(lens) > rows else 0)
        assert m.cu_seqlens_q.tolist() == want and m.cu_seqlens_k.tolist() == [0, lens[0], sum(lens)]
        out = torch.full((rows + 700, hq, d), 3.0, dtype=torch.bfloat16, device=cuda)
        A.prefill_varlen_fp8(q, codes, codes, scales, scales, m.cu_seqlens_q, m.cu_seqlens_k, max(lens), max(lens), 0.1, table, out=out[:rows])
        assert (out[rows:] == 3).all() and (out[:rows] == 0).all()
