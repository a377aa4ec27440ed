"""step_maps on the GPU against lists built token by token."""
import pytest
import torch

from nano_vllm_b200 import _lib
from nano_vllm_b200.step_maps import step_maps
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu


def make(gen, lens, width, free, wide=0):
    """(seq_lens, cached_lens, block_tables [B, width] within rows of width + wide, free_blocks)."""
    seq = torch.tensor([c + n for c, n in lens], dtype=torch.int32)
    cached = torch.tensor([c for c, _ in lens], dtype=torch.int32)
    held = (cached + 255) // 256
    ids = torch.randperm(int(held.sum()) + free, generator=gen).to(torch.int32)
    table = torch.randint(-1, 50, (len(lens), width + wide), generator=gen, dtype=torch.int32)  # leftovers of earlier steps
    at = free
    for b, h in enumerate(held.tolist()):
        table[b, :h] = ids[at:at + h]
        at += h
    return seq, cached, table, ids[:free]


def check(cuda, seq, cached, table, free, rows, width=None, status=0, out=None):
    width = width or table.shape[1]
    dev = table.to(cuda)
    _lib.read_status()
    m = step_maps(seq.to(cuda), cached.to(cuda), dev[:, :width], free.to(cuda), rows, out=out)
    again = step_maps(seq.to(cuda), cached.to(cuda), dev[:, :width], free.to(cuda), rows)
    assert _lib.read_status() == status
    want = F8.step_maps_ref(seq, cached, table[:, :width], free, rows)
    assert dev[:, :width].tolist() == want[0]
    assert torch.equal(dev[:, width:].cpu(), table[:, width:])
    for got in (m, again):
        assert [t.tolist() for t in got[:4]] == [list(x) for x in want[1:5]] and got.blocks_taken.tolist() == [want[5]]
    return m


@pytest.mark.parametrize("lens", [
    [(0, 1)], [(0, 256)], [(0, 257)], [(255, 1)], [(256, 1)], [(300, 0)], [(0, 0)],
    [(0, 0), (3, 5), (0, 0), (0, 0), (256, 256), (511, 2), (0, 0)],
    [(100, 1), (255, 1), (256, 1), (1000, 1)],
])
def test_small_steps(cuda, lens):
    g = torch.Generator().manual_seed(len(lens))
    n = sum(m for _, m in lens)
    seq, cached, table, free = make(g, lens, 6, 9)
    check(cuda, seq, cached, table, free, n)
    check(cuda, seq, cached, table, free, n + 13)


@pytest.mark.parametrize("batch", [31, 256, 257, 1000, 4096])
def test_batches(cuda, batch):
    g = torch.Generator().manual_seed(batch)
    lens = [(int(c), int(n)) for c, n in zip(torch.randint(0, 700, (batch,), generator=g), torch.randint(0, 60, (batch,), generator=g))]
    lens[batch // 2] = (5, 900)
    seq, cached, table, free = make(g, lens, 4, 2 * batch + 8, wide=3)
    check(cuda, seq, cached, table, free, sum(m for _, m in lens) + 5, width=4)


def test_too_few_free_blocks(cuda):
    g = torch.Generator().manual_seed(3)
    lens = [(0, 300), (250, 10), (0, 1000)]
    seq, cached, table, free = make(g, lens, 5, 4)
    m = check(cuda, seq, cached, table, free, 1310)
    assert int(m.blocks_taken) == 7 and (m.slot_mapping[-300:] == -1).all()
    check(cuda, seq, cached, table, free[:0], 1310)


def test_a_long_prompt(cuda):
    g = torch.Generator().manual_seed(4)
    seq, cached, table, free = make(g, [(70, 100000), (0, 3)], 400, 500)
    check(cuda, seq, cached, table, free, 100003)


def test_what_does_not_fit_is_flagged(cuda):
    """A length beyond the table, a negative one, more tokens than rows: cut, flagged, nothing written outside."""
    i32 = dict(dtype=torch.int32, device=cuda)
    table = torch.full((3, 2), 7, **i32)
    _lib.read_status()
    m = step_maps(torch.tensor([600, -5, 10], **i32), torch.tensor([256, 0, 10], **i32), table, torch.arange(5, **i32), 300)
    assert _lib.read_status() == 2
    assert m.cu_seqlens_q.tolist() == [0, 256, 256, 256] and m.cu_seqlens_k.tolist() == [0, 512, 512, 522]
    assert table.tolist() == [[7, 0], [-1, -1], [7, -1]] and int(m.blocks_taken) == 1
    out = [torch.full((n,), 99, **i32) for n in (4, 4, 110)] + [torch.full((110,), 99, dtype=torch.int64, device=cuda), torch.zeros(1, **i32)]
    m = step_maps(torch.tensor([500, 1, 10], **i32), torch.tensor([256, 0, 10], **i32), table, torch.arange(5, **i32), 100,
                  out=[*out[:2], out[2][:100], out[3][:100], out[4]])
    assert _lib.read_status() == 1
    assert m.positions.tolist() == list(range(256, 356)) and m.slot_mapping.tolist() == list(range(100))
    assert (out[2][100:] == 99).all() and (out[3][100:] == 99).all()


def test_captured_and_replayed_with_other_lengths(cuda):
    g = torch.Generator().manual_seed(5)
    lens = [(c, 1) for c in (255, 256, 300, 511)]
    seq, cached, table, free = make(g, lens, 4, 8)
    dev = [t.to(cuda) for t in (seq, cached, table, free)]
    m = step_maps(*dev, 6)  # warm-up, and the graph's tensors
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step_maps(*dev, 6, out=m)
    for k in range(3):
        seq, cached, table, free = make(g, [(c + 100 * k, 1 + (k == 2)) for c, _ in lens[:3]] + [(0, 0)], 4, 8)
        for to, t in zip(dev, (seq, cached, table, free)):
            to.copy_(t)
        graph.replay()
        want = F8.step_maps_ref(seq, cached, table, free, 6)
        assert dev[2].tolist() == want[0] and [t.tolist() for t in m[:4]] == [list(x) for x in want[1:5]]
    assert _lib.read_status() == 0
