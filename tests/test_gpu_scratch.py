"""Decode calls that may run at the same time have scratch of their own: calls on several streams, graphs that are replayed on
several, branches of one graph; over the bf16 cache and the one in 8 bits."""
import gc

import pytest
import torch

from fp8_cases import assert_within, planes_on, random_planes, tables_for
from nano_vllm_b200 import _lib, attention as A, workloads as W
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu


def fp8_call(gen, cuda, lens, hq, hkv, d):
    """A decode whose sequences are cut, and what it has to return."""
    blocks = sum(-(-n // 256) for n in lens)
    planes, tables = random_planes(gen, blocks, hkv, d), tables_for(gen, lens, blocks)
    q, ctx = torch.randn(len(lens), hq, d, generator=gen).bfloat16(), torch.tensor(lens, dtype=torch.int32)
    args = (q.to(cuda), *planes_on(cuda, *planes), ctx.to(cuda), tables.to(cuda), d ** -0.5)
    out = A.decode_paged_fp8(*args)
    assert_within(out, *F8.decode_fp8_ref(q, *planes, ctx, tables, d ** -0.5))
    return (lambda: A.decode_paged_fp8(*args)), out


def bf16_call(cuda, seed, batch, hq, hkv, d):
    c = W.make_decode_case(seed, batch, 500, 3000, hq, hkv, d).to(cuda)
    call = lambda: A.decode_paged(c.q, c.k_cache, c.v_cache, c.context_lens, c.block_tables, c.scale)  # noqa: E731
    return call, call()


@pytest.fixture
def calls(cuda):
    g = torch.Generator().manual_seed(3)
    return [fp8_call(g, cuda, [3000, 20, 900], 16, 8, 128), fp8_call(g, cuda, [1, 4000], 16, 8, 128), fp8_call(g, cuda, [2500] * 5, 14, 2, 64),
            bf16_call(cuda, 1, 4, 16, 8, 128), bf16_call(cuda, 2, 3, 14, 2, 64)]


def captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def test_calls_on_several_streams(cuda, calls):
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [[] for _ in calls]
    for _ in range(60):
        for stream, (call, _), out in zip(streams, calls, outs):
            with torch.cuda.stream(stream):
                out.append(call())
    torch.cuda.synchronize()
    for (_, want), out in zip(calls, outs):
        assert all(torch.equal(o, want) for o in out)
    assert _lib.read_status() == 0


def test_graphs_and_calls_on_several_streams(cuda, calls):
    """All graphs are captured on one stream, as torch does by itself, and replayed on one each, beside calls on another."""
    graphs = [captured(call) for call, _ in calls]
    streams = [torch.cuda.Stream() for _ in range(2 * len(calls))]
    wrong = []
    torch.cuda.synchronize()
    for _ in range(60):
        for k, ((graph, out), (call, want)) in enumerate(zip(graphs, calls)):
            with torch.cuda.stream(streams[2 * k]):
                out.fill_(7)
                graph.replay()
                wrong.append((out != want).sum())
            with torch.cuda.stream(streams[2 * k + 1]):
                wrong.append((call() != want).sum())
    torch.cuda.synchronize()
    assert torch.stack(wrong).sum() == 0
    assert _lib.read_status() == 0


def test_branches_of_one_graph(cuda, calls):
    side = torch.cuda.Stream()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                left = [calls[k][0]() for k in (0, 2, 3)]
            right = [calls[k][0]() for k in (1, 4, 1)]
            torch.cuda.current_stream().wait_stream(side)
        for _ in range(30):
            for o in left + right:
                o.fill_(7)
            graph.replay()
            for o, k in zip(left + right, (0, 2, 3, 1, 4, 1)):
                assert torch.equal(o, calls[k][1])
    assert _lib.read_status() == 0


def test_a_capture_needs_no_call_before_it(cuda):
    """Scratch for a size that no call has had yet, on a stream of its own, is there and zero at the first replay."""
    g = torch.Generator().manual_seed(4)
    call, want = fp8_call(g, cuda, [700, 3, 2000], 64, 8, 128)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        assert torch.equal(out, want)
    with torch.cuda.stream(torch.cuda.Stream()):  # and a stream that has had a smaller one, and none
        small, first = fp8_call(g, cuda, [300], 2, 1, 64)
        assert torch.equal(call(), want) and torch.equal(small(), first) and torch.equal(call(), want)
    torch.cuda.synchronize()
    assert _lib.read_status() == 0


def test_scratch_of_graphs_that_are_gone_is_used_again(cuda, calls):
    held = []
    for k in range(40):
        graph, out = captured(calls[k % len(calls)][0])
        graph.replay()
        assert torch.equal(out, calls[k % len(calls)][1])
        del graph, out
        gc.collect()
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated())
    assert held[-1] <= held[9] + (8 << 20), held  # a buffer has 1 to 3 MB: not one more for every graph
