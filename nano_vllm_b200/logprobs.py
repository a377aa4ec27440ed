"""Log probabilities of tokens: what an engine answers with beside the tokens themselves, and what a search over several
answers goes by.  nano-vllm's ``Sampler`` (nanovllm/layers/sampler.py:10-26) returns tokens only.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from .attention import _native


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # fp32 [N]: of the given tokens
    entropy: torch.Tensor       # fp32 [N]: of the rows' distributions, in nats
    top_tokens: torch.Tensor    # int64 [N, top]: the most probable tokens in order, ties to the lowest index
    top_logprobs: torch.Tensor  # fp32 [N, top]: theirs


class HeadLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32 [N]
    entropy: torch.Tensor   # fp32 [N]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, temperatures: torch.Tensor | None = None,
                   out: Sequence[torch.Tensor] | None = None) -> TokenLogprobs:
    """Under ``softmax(logits / T)`` of every row of ``logits`` ``[N, V]`` (bf16 or fp32): the log probability of its token of
    ``tokens`` (int64 ``[N]``), the entropy, and the ``top`` (0 to 64) most probable tokens with theirs.  One launch, one read
    of the logits; all statistics in fp32.

    ``temperatures``: fp32 ``[N]`` as for ``sample_tokens``, where 1 stands for any that is not above 0 (greedy rows); without
    them T is 1; above 1e30 it counts as 1e30, below 1e-38 as 1e-38.  V is up to 2^24 (2^21 in ``head_logprobs``).  A negative token
    asks for none: 0 (rows of a padded batch); one beyond the vocabulary gives NaN and sets bit 8 of ``_lib.read_status()``.
    Logits of -infinity are masked tokens.  A row with a NaN, with +infinity or with nothing but -infinity has no distribution and
    NaN for results; its ``top_tokens`` go by the logits, NaN like -infinity.
    ``out``: the four result tensors of an earlier call or of a graph, else they are made.  They lie apart from one another and from
    the logits; ``tokens`` and ``temperatures`` may be results' own places (one alternative for each token)."""
    return TokenLogprobs._make(_native(logits).token_logprobs(logits, tokens, top, temperatures, out))


def head_logprobs(hidden_states: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, temperatures: torch.Tensor | None = None,
                  out: Sequence[torch.Tensor] | None = None) -> HeadLogprobs:
    """``token_logprobs`` of ``hidden_states @ weight.T`` (bf16 ``[N, H]`` and ``[V, H]``, H a multiple of 8), without those logits: they
    are summed in fp32, not rounded, and never written.  For scoring what has been given: all positions of a prompt, answers
    of another engine, the reference side of a comparison of two models; nano-vllm computes logits of a prompt's last position only
    (``ParallelLMHead.forward``, nanovllm/layers/embed_head.py:68-88).  Tokens, temperatures and ``out`` (two tensors) as there.

    What the sums lose on average in a tensor core is made good: differences of logits are 1e-7 off on average, relative to
    themselves, where the states' elements are alike, and up to 9.5e-7 too large where a few of them make up the sums, which then
    lose little or nothing."""
    return HeadLogprobs._make(_native(hidden_states).head_logprobs(hidden_states, weight, tokens, temperatures, out))
