"""Attention of a batch whose sequences share prefixes -- several samples of a prompt, requests under one system prompt
-- over a paged cache, on gfx950: the prefix is read and computed once for all sequences of a group, by C ABI
``mi355_shared_prefix_attention_fwd``.

The reference's decode attention (src/kernels/paged_attention_triton.py:23) reads every sequence's whole context.
"""
from __future__ import annotations

import torch

from .. import _lib
from .kv_cache_hip import KVCache

__all__ = ["shared_prefix_attention"]


def shared_prefix_attention(q: torch.Tensor, cache: KVCache, seq_lens: torch.Tensor, prefix_lens: torch.Tensor,
                            groups: torch.Tensor | None = None, *, new_lens: torch.Tensor | None = None,
                            tree_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """``tree_attention`` for a batch whose sequences share prefixes.  Group g -- sequences ``groups[g]`` to ``groups[g
    + 1] - 1`` (int32 [n + 1], ascending); without ``groups``, every batch / n sequences -- shares its first
    ``prefix_lens[g]`` slots (int32 [n]): they are those of the group's first sequence, whatever the page table says of
    the others there.  A sequence with fewer than that in the cache shares what it has; one outside all groups shares
    nothing.

    The other arguments and the result are those of ``tree_attention``: q [batch, tokens, q_heads, head_dim], at most
    ``TREE_ATTENTION_MAX_TOKENS`` new tokens per sequence, which are in the cache already, behind ``seq_lens[b]`` others
    (the prefix among them).

    Where all members' page tables name the prefix's pages, ``tree_attention`` computes the same, and is faster while it
    would read less than about 64 MB of prefixes, once for each member."""
    if scale is None:
        scale = cache.k.shape[-1] ** -0.5
    return _lib.ext().shared_prefix_attention(q, cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale,
                                              seq_lens, prefix_lens, groups, new_lens, tree_mask, scale)
