"""Temperatures close to zero: subnormal ones are above zero, and 1/T is 1e38 at most."""
import pytest
import torch

from nano_vllm_b200.logprobs import head_logprobs, token_logprobs
from oracle.logprobs_ref import assert_same, head_logprobs_ref, logprobs_ref

pytestmark = pytest.mark.gpu
TINY = torch.tensor([1e-39, 1e-45, 1e-38, 1.2e-38, 2e-38, 1e-37, 3e-36, -1e-39, -0.0, 0.0])


def fp32(x):
    return x.float().double()  # what lies beyond fp32 is infinite there


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [37, 40000])
def test_token_logprobs(cuda, dtype, vocab):
    """The largest logit's token has all of a row; rows that are not above zero are untempered."""
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(10, vocab, generator=g) * 3).to(dtype)
    logits[3, 5] = logits[3].max()  # at least two tokens share a row
    tokens = logits.float().argmax(-1)
    tokens[1::4] = (tokens[1::4] + 1) % vocab
    got = token_logprobs(logits.to(cuda), tokens.to(cuda), 4, TINY.to(cuda))
    given, entropy, ids, alternatives, bounds = logprobs_ref(logits, tokens, 4, torch.where(TINY > 0, TINY.double().clamp(min=1e-38), 1.0))
    assert torch.equal(got.top_tokens.cpu(), ids)
    assert_same(got.logprobs, fp32(given), bounds[0], "logprobs")
    assert_same(got.entropy, entropy, bounds[1], "entropy")
    assert_same(got.top_logprobs, fp32(alternatives), bounds[2], "top_logprobs")


@pytest.mark.parametrize("hidden", [64, 1536])
def test_head_logprobs(cuda, hidden):
    g = torch.Generator().manual_seed(hidden)
    w = torch.randn(3001, hidden, generator=g).bfloat16()
    x = torch.randn(10, hidden, generator=g).bfloat16()
    z = x.double() @ w.double().T
    tokens = z.argmax(-1)
    above = TINY > 0
    got = head_logprobs(x.to(cuda), w.to(cuda), tokens.to(cuda), TINY.to(cuda))
    # the largest logit stands apart by far more than the 1e-5 that they may be off: all others' weights are 0
    best = torch.topk(z, 2, dim=-1).values
    assert bool((best[:, 0] - best[:, 1] > 1e-3).all())
    assert not got.logprobs[above.to(cuda)].any() and not got.entropy[above.to(cuda)].any()
    given, entropy, bounds = head_logprobs_ref(x[~above], w, tokens[~above])
    assert_same(got.logprobs[(~above).to(cuda)], given, bounds[0], "logprobs")
    assert_same(got.entropy[(~above).to(cuda)], entropy, bounds[1], "entropy")
