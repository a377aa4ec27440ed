"""Blocks of a cache copied, forked, compacted and listed on the GPU, against lists built entry by entry."""
import pytest
import torch

from nano_vllm_b200 import _lib
from nano_vllm_b200.pages import compact_blocks, copy_blocks, fork_sequences, free_list
from oracle import pages_ref as R

pytestmark = pytest.mark.gpu


def cache(gen, num_blocks, hkv, d, layers, eight=False):
    shape = 2, layers, num_blocks, 256, hkv, d
    if not eight:
        return (torch.randint(-2**15, 2**15, shape, generator=gen, dtype=torch.int16).view(torch.bfloat16),)
    codes = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return codes, torch.rand(2, layers, num_blocks, hkv, 16, generator=gen)


def bits(t):
    return t.contiguous().view(torch.uint8)


def same(got, want):
    return all(torch.equal(bits(a.cpu()), bits(b)) for a, b in zip(got, want))


def sequences(gen, lens, num_blocks, width=None, wide=0, shared=0):
    """(table [B, width] within rows of width + wide as a list and as a tensor, free ids); entries behind a sequence are leftovers."""
    need = [R.blocks_of(n) for n in lens]
    width = width or max(1, *need)
    ids = torch.randperm(num_blocks, generator=gen).tolist()
    table = torch.randint(-5, 2 * num_blocks, (len(lens), width + wide), generator=gen, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        common = min(n, shared, need[b - 1]) if b else 0
        row = table[b - 1, :common].tolist() + ids[at:at + n - common]
        at += n - common
        table[b, :n] = torch.tensor(row, dtype=torch.int32)
    return table[:, :width], ids[at:]


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("hkv,d,layers,eight", [(8, 128, 3, False), (2, 64, 2, False), (8, 128, 2, True), (1, 64, 1, True), (1, 8, 5, False),
                                                (3, 96, 1, False), (5, 16, 7, True)])
def test_copies(cuda, hkv, d, layers, eight):
    g = torch.Generator().manual_seed(hkv * d + layers)
    before = cache(g, 23, hkv, d, layers, eight)
    src = [0, 1, 2, 2, 22, 3, -1, 4, 5, 6, 0, 7]
    dst = [10, 11, 12, 13, 14, 15, 16, -3, 17, 18, 19, 7]
    slots = [256, 0, 1, 15, 16, 17, 256, 256, 255, 1000, -4, 100]
    for given in (slots, None):
        want = tuple(c.clone() for c in before)
        R.copy_ref(want, list(zip(src, dst, given or [256] * len(src))))
        got = tuple(c.to(cuda) for c in before)
        _lib.read_status()
        copy_blocks(got, i32(src, cuda), i32(dst, cuda), None if given is None else i32(given, cuda))
        assert _lib.read_status() == 0 and same(got, want)
    copy_blocks(got, i32([], cuda), i32([], cuda))
    assert same(got, want)
    copy_blocks(got, i32([0, 23, 1], cuda), i32([23, 0, 2**31 - 1], cuda))  # beyond the cache: left out and flagged
    assert _lib.read_status() == 2 and same(got, want)


def test_copies_in_a_cache_of_many_tensors(cuda):
    """One layer's planes at a time, views into an engine's cache, blocks further apart than they are large."""
    g = torch.Generator().manual_seed(5)
    whole, scale = cache(g, 9, 2, 64, 40, True)
    want = whole.clone(), scale.clone()
    R.copy_ref(want, [(1, 4, 40), (8, 0, 256)])
    src, dst, slots = i32([1, 8], cuda), i32([4, 0], cuda), i32([40, 256], cuda)
    got = whole.to(cuda), scale.to(cuda)
    copy_blocks([t[p, layer] for t in got for p in range(2) for layer in range(40)], src, dst, slots)
    assert same(got, want)
    got = whole.to(cuda), scale.to(cuda)
    copy_blocks([t[p] for t in got for p in range(2)], src, dst, slots)
    assert same(got, want)
    wide = torch.zeros(5, 9, 2, 256, 2, 64, dtype=torch.bfloat16, device=cuda)  # K and V of a block side by side
    wide.copy_(torch.randn(wide.shape, generator=g))
    want = wide.cpu()
    for k in range(2):
        R.copy_ref((want[:, :, k],), [(1, 4, 40), (8, 0, 256)])
    copy_blocks([wide[:, :, 0], wide[:, :, 1]], src, dst, slots)
    assert same((wide,), (want,))


def test_copies_beyond_32_bits(cuda):
    """A plane of more than 2^32 bytes, and planes further apart."""
    c = torch.zeros(2, 1, 9000, 256, 8, 128, dtype=torch.bfloat16, device=cuda)
    c[:, :, 8999] = 1.5
    c[:, :, 7] = 2.5
    copy_blocks((c,), i32([8999, 7], cuda), i32([3, 8998], cuda), i32([256, 9], cuda))
    assert bool((c[:, :, 3] == 1.5).all()) and bool((c[:, :, 8998, :9] == 2.5).all()) and not bool(c[:, :, 8998, 9:].any())
    assert not bool(c[:, :, 4:7].any()) and not bool(c[:, :, :3].any())


def check_fork(cuda, gen, lens, parents, eight=False, spare=None, wide=0, status=0, layers=2, hkv=2, d=64):
    need = sum(map(R.blocks_of, lens)) + len(parents)
    num_blocks = max(need, 3)
    table, free = sequences(gen, lens, num_blocks, wide=wide)
    free = free[:spare] if spare is not None else free
    before = cache(gen, num_blocks, hkv, d, layers, eight)
    rows, now, taken, copies = R.fork_ref(table.tolist(), lens, parents, free)
    want = tuple(c.clone() for c in before)
    R.copy_ref(want, copies)
    got = tuple(c.to(cuda) for c in before)
    args = got, table.to(cuda) if not wide else None, i32(lens, cuda), i32(parents, cuda), i32(free, cuda)
    if wide:
        held = torch.zeros(table.shape[0], table.shape[1] + wide, dtype=torch.int32, device=cuda)
        held[:, :table.shape[1]] = table.to(cuda)
        args = got, held[:, :table.shape[1]], *args[2:]
    _lib.read_status()
    for _ in range(2):  # the same call again leaves the same
        f = fork_sequences(*args)
        assert f.block_tables.tolist() == rows and f.seq_lens.tolist() == now and f.blocks_taken.tolist() == [taken]
        assert same(got, want)
    assert _lib.read_status() == status


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lens,parents", [
    ([1], [0]), ([1], [0, 0]), ([256], [0, 0, 0]), ([257], [0, 0]), ([0], [0, 0]), ([300, 5], [1, 1, 0, 1]), ([300, 5], [1]),
    ([700, 512, 0, 255], [3, 3, 2, 1, 1, 0, 0, 0, 3]), ([300, 20], [-1, 0, -7, 0, 1, -1]), ([9, 9, 9], [-1, -1])])
def test_forks(cuda, lens, parents, eight):
    check_fork(cuda, torch.Generator().manual_seed(len(parents)), lens, parents, eight)


def test_forks_of_many(cuda):
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 900, (300,), generator=g).tolist()
    parents = torch.randint(-1, 300, (1000,), generator=g).tolist()
    check_fork(cuda, g, lens, parents, layers=1, hkv=1, d=8, wide=3)
    lens = [3] * 4096
    check_fork(cuda, g, lens, [i // 2 for i in range(4096)], layers=1, hkv=1, d=8)
    check_fork(cuda, g, [5], [0] * 4096, layers=1, hkv=1, d=8)


def test_forks_of_wide_tables(cuda):
    g = torch.Generator().manual_seed(18)
    check_fork(cuda, g, [100_000, 131_072, 77], [0, 1, 1, 0, 2, 2, 0], layers=1, hkv=1, d=8, wide=5)


def test_forks_without_enough_free_blocks(cuda):
    g = torch.Generator().manual_seed(9)
    check_fork(cuda, g, [300, 5], [1, 1, 0, 1, 0], spare=1)
    check_fork(cuda, g, [300, 5], [1, 1, 0, 1, 0], spare=0)


def test_forks_of_what_is_not_there(cuda):
    g = torch.Generator().manual_seed(10)
    check_fork(cuda, g, [300, 5], [2, 1, 0, 2**31 - 1, 1], status=2)       # parents beyond the batch: empty rows
    c = tuple(t.to(cuda) for t in cache(g, 6, 1, 64, 1))
    f = fork_sequences(c, i32([[1], [9], [-1]], cuda), i32([2**31 - 1, 5, 7], cuda), i32([0, 1, 1, 2, 2], cuda), i32([3, 4, 5], cuda))
    assert f.block_tables.tolist() == [[1], [9], [3], [-1], [4]] and f.seq_lens.tolist() == [256, 5, 5, 7, 7]
    assert _lib.read_status() == 2


def check_free(cuda, gen, lens, num_blocks, held=None, shared=0, width=None, wide=0, status=0):
    table, _ = sequences(gen, lens, num_blocks, width, wide, shared)
    dev = torch.zeros(len(lens), table.shape[1] + wide, dtype=torch.int32, device=cuda)
    dev[:, :table.shape[1]] = table.to(cuda)
    _lib.read_status()
    f = free_list(dev[:, :table.shape[1]], i32(lens, cuda), num_blocks, None if held is None else i32(held, cuda))
    counts, free, n = R.free_list_ref(table.tolist(), lens, num_blocks, held)
    assert f.ref_counts.tolist() == counts and f.free_blocks.tolist() == free and f.num_free.tolist() == [n]
    assert _lib.read_status() == status


@pytest.mark.parametrize("lens,num_blocks", [([1], 1), ([0], 1), ([256], 2), ([257, 0, 3], 5), ([2000, 30, 256, 5], 1023), ([5] * 40, 1025),
                                             ([100] * 700, 5000), ([3000] * 300, 4096), ([3000] * 300, 40000), ([700] * 33, 400000)])
def test_free_lists(cuda, lens, num_blocks):
    g = torch.Generator().manual_seed(num_blocks)
    check_free(cuda, g, lens, num_blocks)
    held = torch.randint(-2, 3, (num_blocks,), generator=g).tolist()
    check_free(cuda, g, lens, num_blocks, held, shared=3, width=max(map(R.blocks_of, lens)) + 5, wide=2)


def test_free_list_and_compaction_of_more_entries_than_threads_hold(cuda):
    """Tables whose entries take the cluster several trips."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 5 * 256, (5000,), generator=g).tolist()
    num_blocks = 5000 * 5 + 77
    check_free(cuda, g, lens, num_blocks, width=31, wide=1)
    check_compact(cuda, g, lens, num_blocks, shared=2, layers=1, hkv=1, d=8)


def test_free_list_of_nothing_and_of_what_is_not_there(cuda):
    f = free_list(torch.zeros(0, 4, dtype=torch.int32, device=cuda), i32([], cuda), 3)
    assert f.ref_counts.tolist() == [0, 0, 0] and f.free_blocks.tolist() == [0, 1, 2] and f.num_free.tolist() == [3]
    _lib.read_status()
    f = free_list(i32([[1, -1], [2, 5], [2, 2**31 - 1]], cuda), i32([512, 512, -9], cuda), 3)
    assert f.ref_counts.tolist() == [0, 1, 1] and f.free_blocks.tolist() == [0, -1, -1]
    assert _lib.read_status() == 2


def check_compact(cuda, gen, lens, num_blocks, held=None, shared=0, eight=False, layers=2, hkv=2, d=64, in_place=False):
    table, _ = sequences(gen, lens, num_blocks, shared=shared)
    before = cache(gen, num_blocks, hkv, d, layers, eight)
    now, moved, live, moves = R.compact_ref(table.tolist(), lens, num_blocks, held)
    want = tuple(c.clone() for c in before)
    R.copy_ref(want, [(s, t, 256) for s, t in moves])
    got = tuple(c.to(cuda) for c in before)
    dev = table.to(cuda)
    out = (dev, torch.empty(num_blocks, dtype=torch.int32, device=cuda), torch.empty(1, dtype=torch.int32, device=cuda)) if in_place else None
    _lib.read_status()
    c = compact_blocks(got, dev, i32(lens, cuda), None if held is None else i32(held, cuda), out)
    assert c.block_tables.tolist() == now and c.moved_to.tolist() == moved and c.num_live.tolist() == [live]
    assert same(got, want) and _lib.read_status() == 0
    again = compact_blocks(got, c.block_tables.clone(), i32(lens, cuda),
                           None if held is None else i32([held[moved.index(i)] if i in moved else 0 for i in range(num_blocks)], cuda))
    assert same(got, want)  # what is compact stays
    assert again.block_tables.tolist() == now and again.moved_to.tolist() == [i if i < live else -1 for i in range(num_blocks)]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lens,num_blocks,shared", [([1], 1, 0), ([0, 0], 4, 0), ([300, 700, 0, 256, 1], 40, 2), ([300] * 20, 40, 0),
                                                    ([300] * 20, 41, 1), ([256] * 9, 100, 0)])
def test_compactions(cuda, lens, num_blocks, shared, eight):
    g = torch.Generator().manual_seed(num_blocks)
    check_compact(cuda, g, lens, num_blocks, shared=shared, eight=eight)
    held = (torch.rand(num_blocks, generator=g) < 0.2).int().tolist()
    check_compact(cuda, g, lens, num_blocks, held, shared, eight, in_place=True)


def test_compactions_of_many(cuda):
    g = torch.Generator().manual_seed(3)
    check_compact(cuda, g, [2000] * 300, 9000, layers=1, hkv=1, d=8)
    check_compact(cuda, g, [500] * 1000, 20001, shared=1, layers=1, hkv=1, d=8)


def test_captured(cuda):
    """All four in one graph, replayed on other tables."""
    g = torch.Generator().manual_seed(6)
    lens, num_blocks = [300, 600, 5, 0], 16
    table, free = sequences(g, lens, num_blocks)
    c = cache(g, num_blocks, 2, 64, 2)
    got, dev, n, parents = tuple(t.to(cuda) for t in c), table.to(cuda), i32(lens, cuda), i32([1, 1, 0, 2], cuda)

    def step():
        f = free_list(dev, n, num_blocks)
        k = fork_sequences(got, dev, n, parents, f.free_blocks)
        m = compact_blocks(got, k.block_tables, k.seq_lens)
        copy_blocks(got, i32_src, i32_dst)
        return f, k, m

    i32_src, i32_dst = i32([0, -1], cuda), i32([15, 3], cuda)
    step()
    for t, o in zip(got, c):
        t.copy_(o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f, k, m = step()
    for seed in (1, 2):
        g.manual_seed(seed)
        lens = torch.randint(0, 800, (4,), generator=g).tolist()
        order = torch.randint(-1, 4, (4,), generator=g).tolist()
        table, _ = sequences(g, lens, num_blocks, width=table.shape[1]) if max(lens) <= 768 else sequences(g, [min(n, 700) for n in lens], num_blocks, width=table.shape[1])
        lens = [min(n, 700) for n in lens] if max(lens) > 768 else lens
        for a, b in ((dev, table), (n, torch.tensor(lens)), (parents, torch.tensor(order))):
            a.copy_(b.to(cuda))
        for t, o in zip(got, c):
            t.copy_(o)
        graph.replay()
        counts, free, _ = R.free_list_ref(table.tolist(), lens, num_blocks)
        assert f.ref_counts.tolist() == counts and f.free_blocks.tolist() == free
        rows, now, _, copies = R.fork_ref(table.tolist(), lens, order, free)
        want = tuple(t.clone() for t in c)
        R.copy_ref(want, copies)
        assert k.block_tables.tolist() == rows and k.seq_lens.tolist() == now
        tables, moved, live, moves = R.compact_ref(rows, now, num_blocks)
        R.copy_ref(want, [(s, t, 256) for s, t in moves])
        R.copy_ref(want, [(0, 15, 256)])
        assert m.block_tables.tolist() == tables and m.moved_to.tolist() == moved and m.num_live.tolist() == [live]
        assert same(got, want)


def test_refusals(cuda):
    c = torch.zeros(2, 3, 5, 256, 2, 64, dtype=torch.bfloat16, device=cuda)
    s = torch.zeros(2, 3, 5, 2, 16, device=cuda)
    e, table, lens = i32([0], cuda), i32([[1, 2]], cuda), i32([300], cuda)
    bad = [(ValueError, ()), (RuntimeError, (c.cpu(),)), (RuntimeError, (c.half(),)), (AssertionError, (c[:, :, :, :128],)),
           (AssertionError, (c, s[:, :, :4])), (AssertionError, (s[..., :8],)), (AssertionError, (c[..., :32],)),
           (AssertionError, (c.transpose(0, 1),)), (AssertionError, (c[:, ::2, :0],)), (TypeError, (1,)), (TypeError, 3),
           (RuntimeError, (c.to(torch.float8_e5m2),)), (_lib.NvllmError, (torch.zeros(5, 256, 1, 4, dtype=torch.bfloat16, device=cuda),)),
           (_lib.NvllmError, (c[:, :, :1].expand(2, 3, 5, 256, 2, 64),))]
    for error, caches in bad:
        with pytest.raises(error):
            copy_blocks(caches, e, e)
        with pytest.raises(error):
            fork_sequences(caches, table, lens, e, e)
        with pytest.raises(error):
            compact_blocks(caches, table, lens)
    for error, args in [(RuntimeError, (e.long(), e)), (AssertionError, (e, i32([0, 1], cuda))), (RuntimeError, (e, e.cpu())),
                        (AssertionError, (e, e, i32([1, 2], cuda))), (AssertionError, (table, table))]:
        with pytest.raises(error):
            copy_blocks((c,), *args)
    out = fork_sequences((c,), table, lens, e, e)
    for error, args in [(RuntimeError, (table.long(), lens, e, e)), (AssertionError, (table, i32([1, 2], cuda), e, e)),
                        (AssertionError, (table[0], lens, e, e)), (RuntimeError, (table, lens, e.float(), e)),
                        (_lib.NvllmError, (table, lens, i32([], cuda), e)), (_lib.NvllmError, (table, lens, i32([0] * 4097, cuda), e)),
                        (AssertionError, (table, lens, e, e, (table, *out[1:]))), (ValueError, (table, lens, e, e, out[:2])),
                        (AssertionError, (table, lens, e, e, (out[0], lens, out[2])))]:
        with pytest.raises(error):
            fork_sequences((c,), *args)
    for error, args in [(AssertionError, (table, lens, 0)), (AssertionError, (table, lens, 400001)), (AssertionError, (table, lens, 5, i32([1], cuda))),
                        (RuntimeError, (table.cpu(), lens, 5)), (RuntimeError, (table, lens.cpu(), 5)), (ValueError, (table, lens, 5, None, (e,)))]:
        with pytest.raises(error):
            free_list(*args)
    m = compact_blocks((c,), table, lens)
    for error, args in [(AssertionError, (table, lens, i32([1], cuda))), (ValueError, (table, lens, None, (table,))),
                        (AssertionError, (table, lens, None, (table, m[1], lens))), (AssertionError, (table, lens, m[1], m))]:
        with pytest.raises(error):
            compact_blocks((c,), *args)
