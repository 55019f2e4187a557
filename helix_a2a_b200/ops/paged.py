"""The paged cache of a context-parallel rank: pages and slots of new tokens, and the tokens' way into the cache.

:func:`extend_tables` and :func:`append_kv` run the kernels of ``csrc/paged.cu``; CPU tensors take the oracles of
``reference_math``.  In the reference both belong to vLLM's block manager and attention backends
(``benchmark/sbatch/run_gb200_aiperf_v3.sbatch:95``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _ext, reference_math as rm


class TablePlan(NamedTuple):
    """What :func:`extend_tables` says about a step's new tokens."""

    slots: torch.Tensor        #: int64 [rows]: ``page * page_size + token`` in this rank's cache, -1 where there is none
    positions: torch.Tensor    #: int32 [rows]: position in the sequence (of a tree: committed tokens + depth)
    seq_lens: torch.Tensor     #: int32 [B]: tokens of each sequence that this rank holds, the new ones among them
    draft_lens: torch.Tensor   #: int32 [B]: new ones of these (they are the last)
    mask: torch.Tensor         #: int64 [rows, mask_words]: bit i = the row's token descends from (or is) the i-th new local token
    missing: torch.Tensor      #: int32 [1]: pages that the free list or the table had no room for (at most 2^31 - 1)


def extend_tables(block_table: torch.Tensor, held: torch.Tensor, free_pages: torch.Tensor, free_used: torch.Tensor,
                  ctx_lens: torch.Tensor, q_start: torch.Tensor, *, rows: int, page_size: int,
                  parents: Optional[torch.Tensor] = None, mask_words: int = 1, cp_size: int = 1, cp_rank: int = 0,
                  interleave: int = 1) -> TablePlan:
    """Give the new tokens of every sequence their places in this rank's paged cache, on the device.

    ``q_start [B + 1]``: rows ``q_start[b]`` to ``q_start[b + 1]`` are the new tokens of sequence ``b``, which follow its
    ``ctx_lens [B]`` committed ones (counted over all ranks).  ``q_start[0]`` is 0 and ``rows >= q_start[B]``; rows behind
    ``q_start[B]`` (a captured graph's padding) get slot -1, position 0 and an empty mask.  The token at place ``p`` of its sequence
    belongs to rank ``p // interleave % cp_size`` (``interleave * cp_size`` at most 2^28).  For a tree of drafted tokens ``parents [rows]`` holds the parent of each
    (its number inside the sequence, smaller than the token's own; -1: the last committed token); without it every token follows the
    one before (a call with a tree has at most 2^20 rows).  The mask has ``64 * mask_words`` (at most 256) bits per row; new local tokens beyond that have none, and
    ``mask_words=0`` leaves the mask out (prompts).

    State, updated in place: ``block_table [B, max_pages]`` (this rank's pages), ``held [B]`` (how many of them are valid: a
    sequence keeps the pages of drafted tokens that were not taken) and ``free_used [1]``: ``free_pages[free_used:]`` are free
    and taken in the order of the sequences.  When they run out, or a sequence outgrows ``max_pages``, its last tokens get slot
    -1, ``seq_lens`` counts the others only, and ``missing`` says how many pages there were too few.  All index tensors are int32.
    """
    if not block_table.is_cuda:
        return TablePlan(*rm.extend_tables_reference(block_table, held, free_pages, free_used, ctx_lens, q_start, parents, rows,
                                                     page_size, mask_words, cp_size, cp_rank, interleave))
    return TablePlan(*_ext.ops().extend_tables(block_table, held, free_pages, free_used, ctx_lens, q_start, parents, rows, page_size,
                                               mask_words, cp_size, cp_rank, interleave))


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
              layout: str = "HND") -> None:
    """Write ``k`` / ``v [rows, Hkv, D]`` (views with strides of 16 bytes' multiples are fine) to ``slots [rows]`` of the caches.

    The caches are ``[pages, Hkv, page, D]`` (``layout="HND"``) or ``[pages, page, Hkv, D]`` (``"NHD"``) of the same type, any
    type whose heads' rows are multiples of 16 bytes.  Negative slots (tokens of other ranks) and slots behind the cache are left out.  The
    others have to be distinct, as those of :func:`extend_tables` are: of two rows with one slot either may stay.
    """
    if layout not in ("HND", "NHD"):
        raise ValueError("layout must be 'HND' or 'NHD'")
    if not k.is_cuda:
        rm.append_kv_reference(k, v, k_cache, v_cache, slots, layout == "HND")
        return
    _ext.ops().append_kv(k, v, k_cache, v_cache, slots, layout == "HND")
