"""token_logprobs on the GPU against 64-bit log probabilities, for every way a row can lie, be masked or tie."""
import math

import pytest
import torch

from nano_vllm_b200 import _lib
from nano_vllm_b200.logprobs import TokenLogprobs, token_logprobs
from oracle.logprobs_ref import assert_same, logprobs_ref

pytestmark = pytest.mark.gpu


def check(cuda, logits, tokens, top=0, temperatures=None, status=0, on_gpu=None, **kw):
    _lib.read_status()
    x = logits.to(cuda) if on_gpu is None else on_gpu
    got = token_logprobs(x, tokens.to(cuda), top, None if temperatures is None else temperatures.to(cuda), **kw)
    assert _lib.read_status() == status
    given, entropy, order, alternatives, bounds = logprobs_ref(logits, tokens, top, temperatures)
    assert torch.equal(got.top_tokens.cpu(), order)
    assert_same(got.logprobs, given, bounds[0], "logprobs")
    assert_same(got.entropy, entropy, bounds[1], "entropy")
    assert_same(got.top_logprobs, alternatives, bounds[2], "top_logprobs")
    return got


def some(gen, rows, vocab, dtype=torch.bfloat16, size=3.0):
    return (torch.randn(rows, vocab, generator=gen) * size).to(dtype), torch.randint(vocab, (rows,), generator=gen)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 151936, 20), (3, 151643, 5), (40, 32000, 64), (200, 4099, 8), (700, 1000, 1), (5, 1, 1), (4, 2, 2), (9, 7, 7), (3, 63, 63),
    (2, 64, 64), (6, 65, 64), (7, 2048, 0), (3, 2049, 33), (33, 8191, 64), (2, 16384, 64), (1200, 300, 3), (1, 33000, 64)])
def test_rows(cuda, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows + vocab)
    logits, tokens = some(g, rows, vocab, dtype)
    logits[torch.arange(rows), tokens] += 6 * torch.rand(rows, generator=g).to(dtype)
    check(cuda, logits, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start", range(9))
def test_rows_off_a_16_byte_boundary(cuda, dtype, start):
    """Views of wider rows: what lies before and behind a row is larger than all of it, and counts for nothing."""
    g = torch.Generator().manual_seed(start)
    for vocab in (1, 5, 17, 1001, 9000):
        wide = torch.full((4, vocab + 23), 1e30, dtype=dtype)
        logits, tokens = some(g, 4, vocab, dtype)
        wide[:, start:start + vocab] = logits
        check(cuda, logits, tokens, min(vocab, 12), on_gpu=wide.to(cuda)[:, start:start + vocab])
        wide[:] = math.nan
        wide[:, start:start + vocab] = logits
        check(cuda, logits, tokens, min(vocab, 12), on_gpu=wide.to(cuda)[:, start:start + vocab])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_temperatures_and_tokens(cuda, dtype):
    g = torch.Generator().manual_seed(2)
    logits, tokens = some(g, 14, 5003, dtype)
    t = torch.tensor([0.0, 1.0, 0.5, -1.0, 2.5, 1e-3, 30.0, math.nan, 0.7, 1e30, 1e-30, 1.0, 0.0, 0.1])
    tokens[3], tokens[4], tokens[11] = -1, -2**40, -7
    check(cuda, logits, tokens, 10, t)
    check(cuda, logits, tokens, 0, t)
    tokens[5], tokens[6] = 5003, 2**40
    check(cuda, logits, tokens, 10, t, status=8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 5003, 40000])
def test_masks(cuda, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(dtype).min
    logits, tokens = some(g, 13, vocab, dtype)
    some_kept = torch.randperm(vocab, generator=g)[:7]
    for row, value in ((0, -math.inf), (1, low), (2, -1e30), (3, -1e4)):  # seven tokens allowed
        kept = logits[row, some_kept].clone()
        logits[row] = value
        logits[row, some_kept] = kept
        tokens[row] = some_kept[3]
    logits[4] = -math.inf               # nothing left
    logits[5] = low                     # everything at the lowest value: uniform
    logits[6] = -math.inf
    logits[6, vocab - 1] = low          # one token, at the lowest value
    logits[7, vocab // 2] = math.nan
    logits[8, 3] = math.inf
    logits[9] = math.nan
    logits[10] = 2.0                    # ties everywhere
    logits[11] = -2.0
    logits[11, vocab // 3:vocab // 3 + 30] = -0.0
    logits[11, vocab // 5] = 0.0
    logits[12] = low
    logits[12, vocab // 2:] = low / 2   # far apart below every clamp
    tokens[6], tokens[12] = vocab - 1, vocab - 2
    for top in (0, 1, 20, 50):
        check(cuda, logits, tokens, top)
    tokens[0] = (int(some_kept.max()) + 1) % vocab
    while int(tokens[0]) in some_kept.tolist():
        tokens[0] = (tokens[0] + 1) % vocab
    assert check(cuda, logits, tokens, 3).logprobs[0].item() == -math.inf


@pytest.mark.parametrize("dtype,step", [(torch.bfloat16, 8), (torch.float32, 4)])
@pytest.mark.parametrize("vocab", [20000, 151643])
def test_alternatives_that_one_thread_reads(cuda, dtype, step, vocab):
    """The largest logits at places that fall to few threads, rising and falling rows, rows with many ties at the last place."""
    g = torch.Generator().manual_seed(vocab)
    logits, tokens = some(g, 10, vocab, dtype, size=1.0)
    for row, stride in enumerate((256, 512, 1024, 2048, 4096)):  # threads' strides in pieces
        piece = torch.arange(vocab) // step % stride
        logits[row, piece == 5] += 50
    logits[5] = torch.linspace(-20, 20, vocab).to(dtype)
    logits[6] = torch.linspace(20, -20, vocab).to(dtype)
    logits[7] = (torch.arange(vocab) % 97 < 5).to(dtype) * 4
    logits[8] = torch.randint(0, 3, (vocab,), generator=g).to(dtype)
    logits[9, ::step] += 30
    check(cuda, logits, tokens, 64)
    check(cuda, logits[:7], tokens[:7], 20)


@pytest.mark.parametrize("top", [5, 20, 64])
@pytest.mark.parametrize("rows,vocab", [(3, 743), (150, 1003), (700, 1000), (4, 8000), (2, 40001), (70, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_alternatives_among_ties_and_runs(cuda, dtype, rows, vocab, top):
    """Masks that leave a few tokens here and there, in one place or before the end, equal logits and ones that ascend."""
    g = torch.Generator().manual_seed(vocab + top)
    x, tokens = some(g, rows, vocab, dtype)
    kind = torch.arange(rows) % 6
    few = torch.rand(rows, vocab, generator=g) * vocab < torch.tensor([3.0, 30.0])[torch.arange(rows) % 2][:, None]
    few[:, 5] = True
    x[(kind == 0)[:, None] & ~few] = -torch.inf
    x[(kind == 1)[:, None] & ~few] = torch.finfo(dtype).min
    at = torch.arange(vocab)
    x[kind == 2] = x[kind == 2].masked_fill((at < vocab // 2) | (at > vocab // 2 + 12), -torch.inf)
    x[kind == 3] = x[kind == 3].masked_fill(at < vocab - 9, -torch.inf)
    x[kind == 4] = 1.5
    x[kind == 5] = (at * 0.01).to(dtype)
    tokens[:] = 5
    check(cuda, x, torch.where(torch.isfinite(x[torch.arange(rows), tokens]), tokens, vocab - 1), top)


@pytest.mark.parametrize("dtype,rows,vocab,top", [
    (torch.float32, 300, 33333, 20), (torch.bfloat16, 300, 65536 + 8 * 3 * 256, 20), (torch.bfloat16, 299, 71117, 64), (torch.float32, 160, 66000, 64),
    (torch.float32, 297, 32768 + 4 * 256, 64)])
def test_alternatives_of_threads_with_many_pieces(cuda, dtype, rows, vocab, top):
    """Rows that few threads read: large logits early, late, everywhere, equal and masked ones."""
    g = torch.Generator().manual_seed(vocab)
    x, tokens = some(g, rows, vocab, dtype)
    at, kind = torch.arange(vocab), torch.arange(rows) % 10
    x[kind == 1] = x[kind == 1].masked_fill(torch.rand(vocab, generator=g) < 0.9999, -torch.inf)
    x[kind == 2] = (at * 0.01).to(dtype)
    x[kind == 3] = (at * -0.01).to(dtype)
    x[kind == 4] = x[kind == 4].masked_fill(at < vocab - 5, -torch.inf)
    x[kind == 5] = x[kind == 5].masked_fill(at >= 3, torch.finfo(dtype).min)
    x[kind == 6] = 2.5
    x[(kind == 7)[:, None] & (at % 4096 < 8)] += 20
    x[(kind == 8)[:, None] & (torch.rand(vocab, generator=g) < 0.01)] = math.nan
    tokens[kind == 1] = x[kind == 1].float().argmax(-1)
    tokens[kind == 4], tokens[kind == 5] = vocab - 2, 1
    wide = torch.full((rows, vocab + 3), math.nan, dtype=dtype, device=cuda)
    wide[:, 1:vocab + 1] = x.to(cuda)
    check(cuda, x, tokens, top, on_gpu=wide[:, 1:vocab + 1])
    check(cuda, x, tokens, top)


def test_sizes_of_32_bits(cuda):
    """Rows further apart than 2^31 elements."""
    wide = torch.zeros(3, 1_500_000_000, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(1)
    logits, tokens = some(g, 3, 3001)
    wide[:, -3001:] = logits.to(cuda)
    check(cuda, logits, tokens, 9, on_gpu=wide[:, -3001:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_vocabulary_of_equal_tokens(cuda, dtype):
    logits = torch.zeros(2, 1 << 24, dtype=dtype, device=cuda)
    got = token_logprobs(logits, torch.tensor([5, -1], device=cuda), 64)
    # 2^24 equal weights: every sum is a whole number, ln 2^24 is off by 2^-23 of itself
    want = 24 * math.log(2.0)
    assert got.top_tokens.tolist() == [list(range(64))] * 2
    for value, expected in ((got.logprobs[0], -want), (got.logprobs[1], 0.0), (got.entropy, want), (got.top_logprobs, -want)):
        assert torch.all((value.double() - expected).abs() <= want * 2.0 ** -22)


def test_temperatures_without_a_bound(cuda):
    """Masked tokens have no weight at any temperature, the others one and the same."""
    g = torch.Generator().manual_seed(12)
    logits = torch.randn(6, 3001, generator=g)
    logits[:, 1::2] = -torch.inf
    t = torch.tensor([math.inf, 3e38, 1e36, 1e31, 1e30, 1e29])
    tokens = torch.tensor([0, 2, 1, 4, 6, 8])
    got = token_logprobs(logits.to(cuda), tokens.to(cuda), 5, t.to(cuda))
    given, entropy, ids, alternatives, bounds = logprobs_ref(logits, tokens, 5, t.clamp(max=1e30))
    assert torch.equal(got.top_tokens.cpu(), ids)
    assert_same(got.logprobs, given, bounds[0], "logprobs")
    assert_same(got.entropy, entropy, bounds[1], "entropy")
    assert_same(got.top_logprobs, alternatives, bounds[2], "top_logprobs")


def test_results_go_where_they_are_wanted(cuda):
    """``out``, a captured graph replayed on new logits, and another stream."""
    g = torch.Generator().manual_seed(4)
    (a, tokens), (b, _) = some(g, 6, 3000), some(g, 6, 3000)
    want_a, want_b = (check(cuda, x, tokens, 4) for x in (a, b))
    x, k = a.to(cuda), tokens.to(cuda)
    out = TokenLogprobs(*(torch.full_like(t, 7) for t in want_a))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, k, 4, out=out)
    assert all(i.data_ptr() == j.data_ptr() for i, j in zip(got, out))
    for values, want in ((a, want_a), (b, want_b)):
        x.copy_(values.to(cuda))
        graph.replay()
        assert all(torch.equal(i, j) for i, j in zip(out, want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(20):
            got = token_logprobs(x, k, 4)
    stream.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(got, want_b))
    empty = token_logprobs(x[:0], k[:0], 4)
    assert [tuple(t.shape) for t in empty] == [(0,), (0,), (0, 4), (0, 4)]


def test_refusals(cuda):
    x, k = torch.zeros(2, 100, dtype=torch.bfloat16, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    out = token_logprobs(x, k, 3)
    for error, args in [
            (RuntimeError, (x.half(), k)), (RuntimeError, (x.cpu(), k)), (AssertionError, (x[0], k)), (AssertionError, (x.T, k)),
            (AssertionError, (x, k.int())), (AssertionError, (x, k[:1])), (AssertionError, (x, k.cpu())), (ValueError, (x, k, -1)),
            (ValueError, (x, k, 65)), (ValueError, (x[:, :5], k, 6)), (RuntimeError, (x, k, 3, torch.ones(2))),
            (AssertionError, (x, k, 3, torch.ones(3, device=cuda))), (RuntimeError, (x, k, 3, torch.ones(2, device=cuda).double())),
            (ValueError, (x, k, 3, None, out[:3])), (RuntimeError, (x, k, 2, None, out)), (TypeError, (x, k, 3, None, (1, 2, 3, 4))),
            (RuntimeError, (x, k, 3, None, (*out[:2], out[2].int(), out[3])))]:
        with pytest.raises(error):
            token_logprobs(*args)
    with pytest.raises(_lib.NvllmError):
        token_logprobs(x.expand(2, 100)[:1].expand(2, 100), k, 3)  # rows that lie on one another
