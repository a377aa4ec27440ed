"""Blocks of a K/V cache on the GPU: copied, forked with their sequences, compacted, the free ones listed.

What several answers of one prompt, a beam search or a cache that is to shrink need beside ``step_maps``.  nano-vllm counts
references on the host (``BlockManager``, nanovllm/engine/block_manager.py:26-113), shares whole blocks only and never copies
one.  Here the tables are the truth: a block is free when no table in use names it, so a sequence frees its blocks by leaving
the tables, and ``free_list`` is what ``step_maps`` and ``fork_sequences`` take blocks from.

``caches`` is what the blocks' contents lie in: a sequence of tensors ``[..., blocks, 256, Hkv, D]`` (bf16, or e4m3 codes) and, for
a cache held in 8 bits, its scales ``[..., blocks, Hkv, 16]`` (fp32); the dimensions before ``blocks`` (K and V, layers) are any
that lie at one stride.  The engine's whole cache is ``(runner.kv_cache,)``, after ``plugin.fp8_kv_cache()`` ``(runner.kv_cache,
runner.kv_scale)``; one layer's is ``(layer.k_cache, layer.v_cache)``.  Nothing here synchronises or reads from the device on the
host, so every call can be captured into a graph.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from . import _lib
from .attention import _native


class FreeList(NamedTuple):
    ref_counts: torch.Tensor   # int32 [num_blocks]
    free_blocks: torch.Tensor  # int32 [num_blocks]: ids without a reference in order, -1 behind them
    num_free: torch.Tensor     # int32 [1]


class Fork(NamedTuple):
    block_tables: torch.Tensor  # int32 [rows, W] of the new sequences
    seq_lens: torch.Tensor      # int32 [rows]
    blocks_taken: torch.Tensor  # int32 [1]: how many of the free blocks the copies need


class Compaction(NamedTuple):
    block_tables: torch.Tensor  # int32 [B, W] with the new ids
    moved_to: torch.Tensor      # int32 [num_blocks]: the new id of every live block, -1 of the others
    num_live: torch.Tensor      # int32 [1]: blocks from this id on are free


def _host_of(caches):
    """The extension module, and the caches as a sequence (what can be gone through only once is)."""
    caches = caches if isinstance(caches, (tuple, list)) else tuple(caches)
    return _native(caches[0]) if caches and isinstance(caches[0], torch.Tensor) else _lib.host(), caches


def copy_blocks(caches: Sequence[torch.Tensor], src_blocks: torch.Tensor, dst_blocks: torch.Tensor,
                num_slots: torch.Tensor | None = None) -> None:
    """Block ``dst_blocks[i]`` becomes block ``src_blocks[i]`` (int32 ``[n]``) in all planes of all ``caches``, bit for bit, in one
    launch; with ``num_slots`` (int32 ``[n]``) only its first ``num_slots[i]`` slots, and the scales of their groups of 16.  Pairs with a
    negative block are left out (the padded size of a captured call).  A block that is copied to may be in no other pair."""
    host, caches = _host_of(caches)
    host.copy_blocks(caches, src_blocks, dst_blocks, num_slots)


def fork_sequences(caches: Sequence[torch.Tensor], block_tables: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor,
                   free_blocks: torch.Tensor, out: Sequence[torch.Tensor] | None = None) -> Fork:
    """Sequences that go on from sequences of a batch: row ``i`` of the result is sequence ``parents[i]`` (int32 ``[rows]``) of
    ``block_tables`` (int32 ``[B, W]``) and ``seq_lens`` (int32 ``[B]``, tokens in the cache); a negative parent gives an empty row.  The
    answers of a prompt, or the beams that survive a step.  1 to 4096 rows from up to 4096.

    Whole blocks are shared.  A begun last block stays with its parent's first new row; every other one gets a block of its own, the
    next of ``free_blocks`` (int32 ``[F]``, in order of the rows), with a copy of the slots in use.  More than there are shows in
    ``blocks_taken``; the rows without one have -1 in their tables.  Parents without a new row simply end: their blocks are free
    once the old tables are given up, not before.  One launch; the same call again leaves the same."""
    host, caches = _host_of(caches)
    return Fork._make(host.fork_sequences(caches, block_tables, seq_lens, parents, free_blocks, out))


def free_list(block_tables: torch.Tensor, seq_lens: torch.Tensor, num_blocks: int, held: torch.Tensor | None = None,
              out: Sequence[torch.Tensor] | None = None) -> FreeList:
    """How often the sequences (``block_tables`` int32 ``[B, W]``, ``seq_lens`` int32 ``[B]``) refer to each of the ``num_blocks`` (up to
    400000) blocks of a cache, and which none of them does.  ``held`` (int32 ``[num_blocks]``) counts references from elsewhere, such as
    prefixes that are kept (the sums have to fit 32 bits).  Entries behind a sequence's last block are not looked at, negative ones name no block, and ones
    beyond ``num_blocks`` set bit 2 of ``_lib.read_status()``.  One launch."""
    return FreeList._make(_native(block_tables).free_list(block_tables, seq_lens, num_blocks, held, out))


def compact_blocks(caches: Sequence[torch.Tensor], block_tables: torch.Tensor, seq_lens: torch.Tensor, held: torch.Tensor | None = None,
                   out: Sequence[torch.Tensor] | None = None) -> Compaction:
    """Moves the live blocks (those that ``free_list`` counts a reference of) to the front of the cache: of ``n`` live blocks those
    with an id of ``n`` or more go to the free ids below ``n``, in order, contents and all.  The result's tables name the new ids
    (``out``'s may be ``block_tables`` themselves); what else names blocks (``held``, a prefix cache) goes by ``moved_to``.  Blocks that
    have been moved away keep their contents.  Two launches."""
    host, caches = _host_of(caches)
    return Compaction._make(host.compact_blocks(caches, block_tables, seq_lens, held, out))
