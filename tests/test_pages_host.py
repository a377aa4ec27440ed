"""Blocks of a cache without a GPU: what the entry points refuse, and the oracle's own consistency."""
import ctypes

import pytest
import torch

from nano_vllm_b200 import _lib, pages
from oracle import pages_ref as R

P, P8, NULL = (ctypes.c_void_p(n) for n in (4096, 4104, 0))


def test_there_is_no_cpu_fallback():
    c, i = torch.zeros(2, 256, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: pages.copy_blocks((c,), i, i), lambda: pages.fork_sequences((c,), i.view(1, 1), i, i, i),
                 lambda: pages.free_list(i.view(1, 1), i, 2), lambda: pages.compact_blocks((c,), i.view(1, 1), i)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def parts(**change):
    p = dict(base=4096, planes=6, plane_stride=10 * 65536, block_stride=65536, slot_bytes=256, scale_heads=0)
    p.update(change)
    return (_lib.CachePart * 1)(_lib.CachePart(**p))


CACHE = [
    ({}, -6), ({"base": 0}, -1), ({"base": 4104}, -2), ({"planes": 0}, -3), ({"planes": 70000}, -3), ({"plane_stride": 65536 * 10 + 8}, -2),
    ({"plane_stride": 16}, -3), ({"planes": 1, "plane_stride": 0}, -6), ({"block_stride": 65520}, -3), ({"block_stride": 65544}, -2),
    ({"slot_bytes": 0}, -3), ({"slot_bytes": 8}, -2), ({"slot_bytes": -16}, -3), ({"scale_heads": 8}, -3), ({"scale_heads": -1}, -3),
    ({"slot_bytes": 0, "scale_heads": 8, "block_stride": 512}, -6), ({"slot_bytes": 0, "scale_heads": 8, "block_stride": 496}, -3)]


def usual(change, code):
    if code == -6 and torch.cuda.is_available():
        pytest.skip("would launch")
    return change


@pytest.mark.parametrize("cache,code", CACHE)
def test_caches_that_are_refused(lib, cache, code):
    p = parts(**usual(cache, code))
    assert lib.nvllm_copy_blocks(p, 1, 10, P, P, NULL, 4, None) == code
    assert lib.nvllm_fork_sequences(p, 1, 10, P, 4, 4, P, 2, P, 3, P, 5, P, 4, P, P, None) == code
    assert lib.nvllm_compact_blocks(p, 1, 10, P, 4, 4, P, 2, NULL, P, 4, P, P, P, 4096, None) == code


@pytest.mark.parametrize("change,code", [
    ({"n": 0}, 0), ({"n": -1}, -3), ({"n": 1 << 31}, -3), ({"src": NULL}, -1), ({"dst": NULL}, -1), ({"blocks": 0}, -3), ({"blocks": 1 << 24}, -3),
    ({"num": 0}, -3), ({"num": 161}, -3), ({"parts": None}, -1)])
def test_copy_refuses(lib, change, code):
    a = dict(parts=parts(), num=1, blocks=10, src=P, dst=P, slots=NULL, n=4)
    a.update(change)
    assert lib.nvllm_copy_blocks(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"table": NULL}, -1), ({"lens": NULL}, -1), ({"parents": NULL}, -1), ({"free": NULL}, -1), ({"to": NULL}, -1), ({"to_lens": NULL}, -1),
    ({"taken": NULL}, -1), ({"stride": 3}, -3), ({"to_stride": 3}, -3), ({"width": 0}, -3), ({"batch": -1}, -3), ({"batch": 4097}, -3),
    ({"rows": 0}, -3), ({"rows": 4097}, -3), ({"n_free": -1}, -3), ({"width": 1 << 23, "stride": 1 << 23, "to_stride": 1 << 23}, -3)])
def test_fork_refuses(lib, change, code):
    a = dict(parts=parts(), num=1, blocks=10, table=P, stride=4, width=4, lens=P, batch=2, parents=P, rows=3, free=P, n_free=5, to=P,
             to_stride=4, to_lens=P, taken=P)
    a.update(change)
    assert lib.nvllm_fork_sequences(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({}, -6), ({"table": NULL}, -1), ({"lens": NULL}, -1), ({"counts": NULL}, -1), ({"free": NULL}, -1), ({"n_free": NULL}, -1),
    ({"stride": 3}, -3), ({"width": 0}, -3), ({"batch": -1}, -3), ({"blocks": 0}, -3), ({"blocks": 400001}, -3)])
def test_free_list_refuses(lib, change, code):
    a = dict(table=P, stride=4, width=4, lens=P, batch=2, held=NULL, blocks=10, counts=P, free=P, n_free=P)
    a.update(usual(change, code))
    assert lib.nvllm_free_list(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"table": NULL}, -1), ({"lens": NULL}, -1), ({"to": NULL}, -1), ({"moved": NULL}, -1), ({"live": NULL}, -1), ({"ws": NULL}, -4),
    ({"bytes": 55}, -4), ({"to_stride": 3}, -3), ({"blocks": 400001}, -3), ({"batch": -1}, -3)])
def test_compact_refuses(lib, change, code):
    a = dict(parts=parts(), num=1, blocks=10, table=P, stride=4, width=4, lens=P, batch=2, held=NULL, to=P, to_stride=4, moved=P, live=P,
             ws=P, bytes=56)
    a.update(change)
    assert lib.nvllm_compact_workspace_bytes(10) == 56
    assert lib.nvllm_compact_blocks(*a.values(), None) == code


def test_the_oracle_keeps_what_sequences_hold():
    """Forked and compacted sequences read the tokens that they had."""
    g = torch.Generator().manual_seed(1)
    lens, parents = [300, 5, 512, 0], [0, 0, 2, 1, 1, 1, -1, 3]
    table = [[7, 3, -1], [1, -1, -1], [0, 11, -1], [-1, -1, -1]]
    c = (torch.randint(-2**15, 2**15, (2, 1, 20, 256, 1, 8), generator=g, dtype=torch.int16).view(torch.bfloat16),)

    def tokens(cache, row, n):
        at = torch.tensor([row[t // 256] * 256 + t % 256 for t in range(n)], dtype=torch.long)
        return cache[0].view(torch.int16).view(2, -1, 8)[:, at]

    had = [tokens(c, table[p], lens[p]) if p >= 0 else tokens(c, [], 0) for p in parents]
    _, free, n = R.free_list_ref(table, lens, 20)
    assert n == 15
    rows, now, taken, copies = R.fork_ref(table, lens, parents, free)
    assert taken == 3 and len({row[1] for row in rows[:2]}) == 2
    R.copy_ref(c, copies)
    assert all(torch.equal(tokens(c, row, m), h) for row, m, h in zip(rows, now, had))
    rows, moved, live, moves = R.compact_ref(rows, now, 20)
    R.copy_ref(c, [(s, t, 256) for s, t in moves])
    assert live == 8 and sorted(i for i in moved if i >= 0) == list(range(8))
    assert all(torch.equal(tokens(c, row, m), h) for row, m, h in zip(rows, now, had))
