"""A paged key/value cache, quantised as it is written, on gfx950.

``KVCache`` holds the tensors: a pool of pages for keys and one for values --
16-bit values, or int8 / e4m3 codes with an fp32 scale per token and head --
and the page table of the sequences at hand.  ``kv_cache_append`` writes new
tokens (rotating queries and keys on the way), ``kv_cache_read`` returns a
range as 16-bit values, ``kv_cache_keep`` moves the accepted tokens of a draft
together, and ``tree_attention`` (tree_attention_hip.py) attends over it.  C
ABI ``mi355_kv_cache_{append,read,keep}_fwd``.

The reference keeps its paged cache in 16 bits (src/kv_cache/block_manager.py);
the codes halve what a decode step reads of it.
"""
from __future__ import annotations

import torch

from .. import _lib

__all__ = ["KVCache", "kv_cache_append", "kv_cache_read", "kv_cache_keep", "KV_FORMATS"]

# name -> storage dtype (None: the model's 16-bit dtype)
KV_FORMATS = {"16bit": None, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class KVCache:
    """The tensors of a paged cache.

    k, v: [pages, kv_heads, page_size, head_dim], contiguous: fp16 / bf16 values
    or int8 / float8_e4m3fn codes.  k_scale, v_scale: float32 [pages, kv_heads,
    page_size] for codes (value = code * scale), None for values.  page_table:
    int32 [batch, n]: slot s of sequence b lies on page ``page_table[b, s //
    page_size]`` at place ``s % page_size``; a page number outside the pool (-1,
    say) marks slots without a place: they are not written, read as zero and are
    not attended to.  page_size is a multiple of 16, head_dim a multiple of 16
    and at most 256.  The object only names the tensors; a batch of other
    sequences over the same pools is another ``KVCache`` with its page table."""

    __slots__ = ("k", "v", "page_table", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        self.k, self.v, self.page_table, self.k_scale, self.v_scale = k, v, page_table, k_scale, v_scale

    @classmethod
    def allocate(cls, batch: int, max_len: int, kv_heads: int, head_dim: int, kv_format: str = "int8",
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cuda",
                 page_size: int | None = None, pages: int | None = None) -> "KVCache":
        """An empty cache of ``max_len`` slots (rounded up to whole pages) for
        each of ``batch`` sequences, its pages in order; one page per sequence
        without ``page_size``.  With ``pages``, a pool of that many and a table
        without any, which ``kv_cache_reserve`` hands out.  kv_format: "16bit" (of
        ``dtype``), "int8" or "e4m3"."""
        if kv_format not in KV_FORMATS:
            raise ValueError(f"unknown kv_format {kv_format!r} ({', '.join(KV_FORMATS)})")
        if page_size is None:
            page_size = max(16, -(-max_len // 16) * 16)
        if page_size < 16 or page_size % 16 or head_dim % 16 or not 0 < head_dim <= 256:
            raise ValueError("page_size and head_dim must be multiples of 16, head_dim at most 256 "
                             f"(got {page_size}, {head_dim})")
        per = max(1, -(-max_len // page_size))
        if pages is not None and pages < 1:
            raise ValueError(f"a pool has at least one page, got {pages}")
        shape = (batch * per if pages is None else pages, kv_heads, page_size, head_dim)
        quantised = kv_format != "16bit"
        pools = [torch.zeros(shape, dtype=torch.uint8 if quantised else dtype, device=device) for _ in range(2)]
        if quantised:
            pools = [p.view(KV_FORMATS[kv_format]) for p in pools]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) if quantised else None for _ in range(2)]
        if pages is None:
            table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        else:
            table = torch.full((batch, per), -1, dtype=torch.int32, device=device)
        return cls(*pools, table, *scales)

    @property
    def capacity(self) -> int:
        """Slots of each sequence that the page table can name."""
        return self.page_table.shape[1] * self.k.shape[2]

    def num_bytes(self) -> int:
        """Bytes of the pools and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def tensors(self) -> tuple:
        return self.k, self.v, self.page_table, self.k_scale, self.v_scale


def kv_cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, seq_lens: torch.Tensor, *,
                    new_lens: torch.Tensor | None = None, q: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
                    scale: float = 1.0, interleaved: bool = False) -> torch.Tensor | None:
    """Writes k, v [batch, tokens, kv_heads, head_dim] (fp16 or bf16, any
    strides) into slots ``seq_lens[b] + t`` (int32 [batch]: tokens in the cache
    before).  Tokens from ``new_lens[b]`` on are padding and not written.  With
    ``positions`` and ``inv_freq`` (see ``fused_rotary``) keys are rotated
    first -- in fp32, without a rounding before the quantisation -- and so is
    ``q`` [batch, tokens, q_heads, head_dim], whose rotation is returned.

    Per token and head, ``scale = max(max|x| / top, 1e-8)`` and ``code = round(x
    / scale)``, top = 127 (int8, ties to even) or 448 (e4m3).  A row that holds
    an infinity or a NaN reads back as NaN."""
    return _lib.ext().kv_append(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, k, v, seq_lens,
                                new_lens, q, positions, inv_freq, scale, interleaved)


def kv_cache_read(cache: KVCache, end: torch.Tensor, tokens: int, *, start: torch.Tensor | None = None,
                  dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of slots ``start[b] + i`` (0 without ``start``), i <
    ``tokens``, as [batch, kv_heads, tokens, head_dim] in ``dtype`` (fp16 / bf16;
    by default the cache's own, fp16 for codes); zeros from slot ``end[b]`` on.
    start and end: int32 [batch]."""
    if dtype is None:
        dtype = cache.k.dtype if cache.k_scale is None else torch.float16
    return _lib.ext().kv_read(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, end, tokens, start,
                              dtype)


def kv_cache_keep(cache: KVCache, seq_lens: torch.Tensor, kept: torch.Tensor,
                  kept_lens: torch.Tensor | None = None) -> None:
    """Moves the kept tokens of a draft together: slot ``seq_lens[b] + i`` becomes
    what slot ``seq_lens[b] + kept[b, i]`` held, for i < ``kept_lens[b]`` (without
    it: all).  kept: int32 [batch, n], n <= 128, in any order; a negative entry
    leaves its slot as it was."""
    _lib.ext().kv_keep(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, seq_lens, kept, kept_lens)
