"""Block tables, slot map, positions and offsets of a step, built on the GPU from the requests' lengths.

The device side of what nano-vllm's ``ModelRunner`` builds in Python for every step, token by token
(``prepare_prefill`` / ``prepare_decode`` / ``prepare_block_tables``, nanovllm/engine/model_runner.py:151-249), for
engines that keep lengths and tables on the GPU: two integers a request go in, and everything that ``store_kvcache``,
``prefill_varlen``, ``decode_paged``, their 8-bit forms and ``qk_norm_rope_store`` are told about the step comes out.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from .attention import _native


class StepMaps(NamedTuple):
    cu_seqlens_q: torch.Tensor  # int32 [B + 1]: offsets of the sequences' new tokens, no more than num_tokens
    cu_seqlens_k: torch.Tensor  # int32 [B + 1]: and of all their tokens
    slot_mapping: torch.Tensor  # int32 [num_tokens]: cache slot of every new token, -1 behind the last one
    positions: torch.Tensor     # int64 [num_tokens]: its position in its sequence, 0 behind the last one
    blocks_taken: torch.Tensor  # int32 [1]: how many of the free blocks the step needs


def step_maps(seq_lens: torch.Tensor, cached_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
              num_tokens: int, out: Sequence[torch.Tensor] | None = None) -> StepMaps:
    """Sequence b has ``cached_lens[b]`` tokens in the cache and ``seq_lens[b]`` with this step (int32 ``[B]``); the first
    ``ceil(cached / 256)`` entries of ``block_tables[b]`` (int32 ``[B, W]``) are its blocks so far.  In place: the entries up
    to ``ceil(seq / 256)`` are taken from ``free_blocks`` in order, sequence after sequence, those behind become -1.
    ``num_tokens``: the step's new tokens, or more (the padded size of a captured batch).

    More blocks needed than there are free shows in ``blocks_taken``; entries without a block are -1 and the slots in them
    too, so nothing is stored there.  ``out``: the five result tensors of an earlier call or of a graph, else they are made.
    One launch, no synchronisation; the same call again leaves the same."""
    return StepMaps._make(_native(seq_lens).step_maps(seq_lens, cached_lens, block_tables, free_blocks, num_tokens, out))
