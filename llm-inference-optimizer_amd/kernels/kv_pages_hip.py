"""Page tables and slot maps made on the GPU from the lengths of requests, on gfx950.

``kv_cache_reserve`` gives the sequences of a ``KVCache`` the pages that their lengths ask for and takes back those that
they do not need any more; ``kv_slot_map`` says where the tokens of a packed batch lie.  Neither looks at a value on
the host, so a captured decode step can grow its sequences page by page.  C ABI ``mi355_kv_cache_reserve_fwd`` and
``mi355_kv_slot_map_fwd``.

The reference allocates the blocks of its paged cache on the host (src/kv_cache/block_manager.py).
"""
from __future__ import annotations

import torch

from .. import _lib
from .kv_cache_hip import KVCache

__all__ = ["kv_cache_reserve", "kv_slot_map"]


def kv_cache_reserve(cache: KVCache, seq_lens: torch.Tensor, new_lens: torch.Tensor | None = None, *,
                     out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages for the slots below ``seq_lens[b] + new_lens[b]`` of every sequence (int32 [batch]; without ``new_lens``:
    below ``seq_lens[b]``; negative numbers count as 0).  Returns (table, missing): the page table, written to ``out``
    (int32 of its shape) or in place, and how many pages each sequence did not get (int32 [batch], 0 where all is well),
    because the pool has no more or the table is too narrow for them.

    Entries that a sequence needs and has stay as they are, those beyond its need become -1.  Free are all pages of the
    pool that no entry which stays names: rows may share pages (copy the entries of a common prefix from row to row),
    and a sequence that ended gives its pages back with a length of 0.  Free pages are handed out in ascending order,
    sequence by sequence.  The table is the only state, so every sequence with tokens in the pool has to have its row
    in it: pages that only another table names count as free."""
    return _lib.ext().kv_reserve(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, seq_lens, new_lens,
                                 out)


def kv_slot_map(cache: KVCache, seq_lens: torch.Tensor, new_lens: torch.Tensor,
                tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Where the new tokens of a packed batch (``new_lens[0]`` tokens of sequence 0, then those of sequence 1, ...;
    int32 [batch], negative numbers count as 0) go.  Returns, for each of ``tokens`` rows:

    * slots (int64): ``page * page_size + place`` of token ``seq_lens[b] + t`` of its sequence, that is ``cache.k[slot //
      page_size, :, slot % page_size]``; -1 without a page
    * sequences (int32): its sequence b
    * positions (int64): ``seq_lens[b] + t``, as ``fused_rotary`` takes them

    Rows behind the last token get -1, -1 and 0; of tokens beyond ``tokens`` nothing is written."""
    return _lib.ext().kv_slot_map(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, seq_lens, new_lens,
                                  tokens)
