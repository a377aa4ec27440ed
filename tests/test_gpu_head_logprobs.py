"""head_logprobs on the GPU against 64-bit log probabilities of the product."""
import math

import pytest
import torch

from nano_vllm_b200 import _lib
from nano_vllm_b200.logprobs import HeadLogprobs, head_logprobs, token_logprobs
from oracle.logprobs_ref import assert_same, head_logprobs_ref

pytestmark = pytest.mark.gpu


def some(gen, rows, hidden, vocab):
    w = (torch.randn(vocab, hidden, generator=gen) * (2.5 / math.sqrt(hidden))).bfloat16()
    tokens = torch.randint(vocab, (rows,), generator=gen)
    x = torch.randn(rows, hidden, generator=gen) + 2 * torch.rand(rows, 1, generator=gen) * w[tokens].float()
    return x.bfloat16(), w, tokens


def check(cuda, x, w, tokens, temperatures=None, status=0, on_gpu=None):
    _lib.read_status()
    a, b = (x.to(cuda), w.to(cuda)) if on_gpu is None else on_gpu
    got = head_logprobs(a, b, tokens.to(cuda), None if temperatures is None else temperatures.to(cuda))
    assert _lib.read_status() == status
    given, entropy, bounds = head_logprobs_ref(x, w, tokens, temperatures)
    assert_same(got.logprobs, given, bounds[0], "logprobs")
    assert_same(got.entropy, entropy, bounds[1], "entropy")
    return got


@pytest.mark.parametrize("rows,hidden,vocab", [
    (1, 64, 1000), (1, 8, 1), (3, 8, 7), (5, 72, 127), (128, 128, 128), (129, 64, 257), (2, 1024, 4000), (1, 1032, 3000), (7, 2048, 2111),
    (40, 896, 5003), (300, 200, 3000), (1000, 64, 1003), (2, 4096, 300), (130, 2056, 900), (257, 1024, 2000), (5, 5120, 640), (1, 64, 38000)])
def test_shapes(cuda, rows, hidden, vocab):
    g = torch.Generator().manual_seed(rows + hidden + vocab)
    check(cuda, *some(g, rows, hidden, vocab))


@pytest.mark.parametrize("rows", [1, 127, 200, 385, 650])
def test_many_tiles(cuda, rows):
    """More tiles than multiprocessors, with row tiles that divide them and that do not."""
    g = torch.Generator().manual_seed(rows)
    check(cuda, *some(g, rows, 128, 30011))


def test_more_row_tiles_than_multiprocessors(cuda):
    g = torch.Generator().manual_seed(1)
    check(cuda, *some(g, 148 * 256 + 130, 16, 700))


def test_rows_whose_statistics_are_kept_for_several_tiles(cuda):
    """So many rows that column tiles go in groups; rows from everywhere against the reference."""
    g = torch.Generator().manual_seed(8)
    x, w, tokens = some(g, 150_000, 16, 5003)
    got = head_logprobs(x.to(cuda), w.to(cuda), tokens.to(cuda))
    rows = torch.cat([torch.arange(3), torch.randint(150_000, (300,), generator=g), torch.arange(149_990, 150_000)])
    given, entropy, bounds = head_logprobs_ref(x[rows], w, tokens[rows])
    assert_same(got.logprobs[rows.to(cuda)], given, bounds[0], "logprobs")
    assert_same(got.entropy[rows.to(cuda)], entropy, bounds[1], "entropy")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("hidden", [64, 1536])
def test_temperatures_tokens_and_strides(cuda, hidden):
    g = torch.Generator().manual_seed(2)
    x, w, tokens = some(g, 14, hidden, 3001)
    t = torch.tensor([0.0, 1.0, 0.5, -1.0, 2.5, 1e-2, 30.0, math.nan, 0.7, 1e30, 1.0, 1.0, 0.0, 0.1])
    tokens[3], tokens[4], tokens[11], tokens[12] = -1, -2**40, 3000, 0
    wide_x = torch.full((14, hidden + 24), math.nan, dtype=torch.bfloat16, device=cuda)
    wide_w = torch.full((3001, hidden + 8), math.nan, dtype=torch.bfloat16, device=cuda)
    wide_x[:, 16:16 + hidden], wide_w[:, 8:] = x.to(cuda), w.to(cuda)
    views = wide_x[:, 16:16 + hidden], wide_w[:, 8:]
    check(cuda, x, w, tokens, t, on_gpu=views)
    check(cuda, x, w, tokens, on_gpu=views)
    tokens[5], tokens[6] = 3001, 2**40
    check(cuda, x, w, tokens, t, status=8, on_gpu=views)


@pytest.mark.parametrize("hidden", [64, 1536])
def test_rows_without_a_distribution(cuda, hidden):
    """NaN and infinities in a row's state stay in that row; rows of zeros are uniform."""
    g = torch.Generator().manual_seed(3)
    x, w, tokens = some(g, 140, hidden, 1500)
    x[1, 3], x[5, 0], x[130, 7], x[2] = math.nan, math.inf, -math.inf, 0
    got = head_logprobs(x.to(cuda), w.to(cuda), tokens.to(cuda))
    broken = [1, 5, 130]
    assert all(torch.isnan(t[broken]).all() for t in got)
    kept = [r for r in range(140) if r not in broken]
    given, entropy, bounds = head_logprobs_ref(x[kept], w, tokens[kept])
    assert_same(got.logprobs[kept], given, bounds[0], "logprobs")
    assert_same(got.entropy[kept], entropy, bounds[1], "entropy")
    assert abs(got.entropy[2].item() - math.log(1500)) < 1e-5


@pytest.mark.parametrize("hidden", [8, 64, 1024, 2056])
def test_sums_of_one_product(cuda, hidden):
    """Products that no sum cuts: what makes good the mean loss of long sums stays within the bound here too."""
    g = torch.Generator().manual_seed(hidden)
    _, w, tokens = some(g, 130, hidden, 700)
    x = torch.zeros(130, hidden)
    x[torch.arange(130), torch.randint(hidden, (130,), generator=g)] = 4.0
    check(cuda, x.bfloat16(), w, tokens)


def test_agrees_with_the_logits_that_it_does_not_write(cuda):
    g = torch.Generator().manual_seed(4)
    x, w, tokens = some(g, 33, 512, 9001)
    a, b, k = x.to(cuda), w.to(cuda), tokens.to(cuda)
    got, from_logits = head_logprobs(a, b, k), token_logprobs(a.float() @ b.float().T, k)
    _, _, bounds = head_logprobs_ref(x, w, tokens)
    assert_same(got.logprobs, from_logits.logprobs.cpu(), 2 * bounds[0], "logprobs")
    assert_same(got.entropy, from_logits.entropy.cpu(), 2 * bounds[1], "entropy")


def test_results_go_where_they_are_wanted(cuda):
    """``out``, a captured graph replayed on other states, two streams at once, and the same bits every time."""
    g = torch.Generator().manual_seed(5)
    x, w, tokens = some(g, 200, 256, 5000)
    y, _, _ = some(g, 200, 256, 5000)
    a, b, k = x.to(cuda), w.to(cuda), tokens.to(cuda)
    want_x, want_y = head_logprobs(a, b, k), head_logprobs(y.to(cuda), b, k)
    out = HeadLogprobs(*(torch.full_like(t, 7) for t in want_x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        head_logprobs(a, b, k, None, out)
    for values, want in ((x, want_x), (y, want_y)):
        a.copy_(values.to(cuda))
        graph.replay()
        assert all(torch.equal(i, j) for i, j in zip(out, want))
    streams, z = [torch.cuda.Stream() for _ in range(2)], [x.to(cuda), y.to(cuda)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(15):
        for s, v, r in zip(streams, z, got):
            with torch.cuda.stream(s):
                r.append(head_logprobs(v, b, k))
    torch.cuda.synchronize()
    for r, want in zip(got, (want_x, want_y)):
        assert all(torch.equal(i, j) for t in r for i, j in zip(t, want))
    assert [tuple(t.shape) for t in head_logprobs(a[:0], b, k[:0])] == [(0,), (0,)]
    assert _lib.read_status() == 0


def test_refusals(cuda):
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(100, 64, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(2, dtype=torch.int64, device=cuda)
    out = head_logprobs(x, w, k)
    for error, args in [
            (RuntimeError, (x.float(), w, k)), (RuntimeError, (x, w.float(), k)), (RuntimeError, (x, w.cpu(), k)), (AssertionError, (x, w[:, :32], k)),
            (AssertionError, (x[0], w, k)), (AssertionError, (x, w, k[:1])), (AssertionError, (x, w, k.int())), (AssertionError, (x.T, x.T, k)),
            (_lib.NvllmError, (x[:, :60], w[:, :60], k)), (_lib.NvllmError, (x[:, 4:60], w[:, :56], k)), (RuntimeError, (x, w, k, torch.ones(2))),
            (_lib.NvllmError, (x, w[:0], k)), (ValueError, (x, w, k, None, out[:1])), (RuntimeError, (x, w, k, None, (out[0], k)))]:
        with pytest.raises(error):
            head_logprobs(*args)
