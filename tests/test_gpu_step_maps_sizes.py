"""step_maps at sizes where a launch's resources change."""
import subprocess
import sys
from pathlib import Path

import pytest

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
