"""Attention of a few new tokens per sequence over a paged cache, on gfx950.

``tree_attention`` is the attention of a decode step (one new token) and of the
verification of drafted tokens: a chain, or a tree of them by ``tree_mask``.
The reference's decode attention (src/kernels/paged_attention_triton.py:23)
takes single queries over a 16-bit cache.  C ABI ``mi355_tree_attention_fwd``.
"""
from __future__ import annotations

import torch

from .. import _lib
from .kv_cache_hip import KVCache

__all__ = ["tree_attention", "TREE_ATTENTION_MAX_TOKENS"]

# New tokens per sequence that the kernel takes.
TREE_ATTENTION_MAX_TOKENS = 128


def tree_attention(q: torch.Tensor, cache: KVCache, seq_lens: torch.Tensor, *, new_lens: torch.Tensor | None = None,
                   tree_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """q: [batch, tokens, q_heads, head_dim] (fp16 or bf16, any strides), tokens
    <= ``TREE_ATTENTION_MAX_TOKENS``; query head h reads key/value head ``h //
    (q_heads // kv_heads)``.  The new tokens' keys and values are in the cache
    already, in slots ``seq_lens[b] + t`` (``kv_cache_append``).  Token t sees all
    slots below ``seq_lens[b]`` and new token j where ``tree_mask`` (bool [tokens,
    tokens] or [batch, tokens, tokens]) is set; without a mask, every j <= t.
    scale: head_dim ** -0.5 by default.

    Returns softmax(scale * q K^T) V as [batch, tokens, q_heads, head_dim], fp32
    sums and one rounding to q's dtype.  Slots that a token does not see have no
    influence, whatever they hold; an infinite 16-bit value that it sees
    makes its element infinite, however small its weight, and a scale of codes
    that is not finite makes all of its elements NaN.  A token that sees nothing, and padding (t >=
    ``new_lens[b]``), gets zeros."""
    if scale is None:
        scale = cache.k.shape[-1] ** -0.5
    return _lib.ext().tree_attention(q, cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, seq_lens,
                                     new_lens, tree_mask, scale)
