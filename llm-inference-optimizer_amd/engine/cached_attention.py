"""Attention blocks that keep their keys and values in a paged, optionally
quantised cache (``KVCache``) and attend over it with the package's kernels.

``CachedAttention`` takes the place of a decoder layer's attention module
(``patch_model_with_fused_kernels(..., fuse_attention=True)``) and reuses its
projections.  Called with a ``DecoderCache``, which ``GraphedGreedyDecoder``
passes as ``past_key_values``, it runs

    q, k, v projections -> kv_cache_append (rotary of q and k, quantisation,
    one kernel) -> tree_attention over the cache -> output projection

and, for a prompt of more tokens than ``tree_attention`` takes, torch's causal
attention over the keys and values read back from the cache, so that the prompt
sees what later tokens will see.  Called with any other cache (or none) it runs
the original module's forward, unchanged.

The reference's engines do this with a 16-bit block cache and single-query
attention (src/engine/paged_engine.py:124-145).
"""
from __future__ import annotations

import torch

from ..kernels.kv_cache_hip import KVCache, kv_cache_append, kv_cache_keep, kv_cache_read
from ..kernels.shared_prefix_hip import shared_prefix_attention
from ..kernels.tree_attention_hip import TREE_ATTENTION_MAX_TOKENS, tree_attention

__all__ = ["CachedAttention", "DecoderCache", "ATTENTION_CLASS_NAMES"]

ATTENTION_CLASS_NAMES = {"Qwen2Attention", "LlamaAttention", "MistralAttention"}
_PARTS = ("q_proj", "k_proj", "v_proj", "o_proj", "head_dim", "layer_idx", "scaling")


class DecoderCache:
    """What a decode step needs to know of the cache, for ``CachedAttention``:
    one ``KVCache`` per layer (they share a page table) and the step's static
    tensors -- ``lens`` (tokens in the cache, int32 [batch]), ``positions`` (of
    the step's tokens, int64 [batch, tokens]), ``new_lens`` and ``tree_mask`` (None,
    or of a draft).  HF's forward sees an empty cache of its own kind through
    ``as_past()``: it builds no buffers for it.

    ``shared_prefix`` (None, or int32 [groups]): every batch / groups sequences share
    that many of their first slots, which ``shared_prefix_attention`` then reads and
    computes once for all of them.

    ``prompt``: the cache is empty before the step, which may then have more tokens
    than ``tree_attention`` takes.

    What a token sees is said by these tensors alone: a padded batch, or any
    attention mask but a causal one, is refused (padding goes behind a row's
    tokens, with ``new_lens``).  ``unmasked``: set by a caller that passes the model
    no mask, so that the one that HF may build needs no look, which waits for the
    GPU."""

    def __init__(self, layers: list[KVCache], inv_freq: torch.Tensor, rotary_scale: float):
        self.layers = layers
        self.inv_freq = inv_freq
        self.rotary_scale = rotary_scale
        batch = layers[0].page_table.shape[0]
        self.lens = torch.zeros((batch,), dtype=torch.int32, device=layers[0].k.device)
        self.positions = self.new_lens = self.tree_mask = self.shared_prefix = None
        self.prompt = self.unmasked = False

    @classmethod
    def allocate(cls, model, batch_size: int, max_len: int, kv_format: str, page_size: int | None = None,
                 pages: int | None = None):
        """For an HF causal LM whose attention modules are ``CachedAttention``.  pages: as in ``KVCache.allocate``."""
        blocks = [layer.self_attn for layer in model.model.layers]
        if not all(isinstance(b, CachedAttention) for b in blocks):
            raise ValueError("kv_cache needs the model's attention patched: "
                             "patch_model_with_fused_kernels(model, fuse_attention=True)")
        rotary = model.model.rotary_emb
        if getattr(rotary, "rope_type", "default") in ("dynamic", "longrope"):
            raise ValueError(f"rope_type {rotary.rope_type!r} changes the frequencies as the text grows: cached keys "
                             "would keep old ones")
        p = next(model.parameters())
        layers = [KVCache.allocate(batch_size, max_len, b.k_proj.out_features // b.head_dim, b.head_dim, kv_format,
                                   p.dtype, p.device, page_size, pages) for b in blocks]
        table = layers[0].page_table
        for c in layers:
            c.page_table = table
        return cls(layers, rotary.inv_freq.to(device=p.device, dtype=torch.float32), float(rotary.attention_scaling))

    def as_past(self):
        """An HF cache object that carries this one."""
        from transformers import DynamicCache

        past = DynamicCache()
        past.mi355_cache = self
        return past

    def keep(self, kept: torch.Tensor, kept_lens: torch.Tensor) -> None:
        """``kv_cache_keep`` in every layer."""
        for c in self.layers:
            kv_cache_keep(c, self.lens, kept, kept_lens)

    def num_bytes(self) -> int:
        return sum(c.num_bytes() for c in self.layers)


def cacheable(module: torch.nn.Module) -> bool:
    """Whether ``CachedAttention`` can run this attention module: grouped heads
    of a width the cache takes, no window and no norms of queries and keys."""
    # a module without a window of its own may take the model's
    config = getattr(module, "config", None)
    window = module.sliding_window if hasattr(module, "sliding_window") else getattr(config, "sliding_window", None)
    return (module.__class__.__name__ in ATTENTION_CLASS_NAMES and all(hasattr(module, p) for p in _PARTS)
            and window is None and not hasattr(module, "q_norm")
            and module.head_dim % 16 == 0 and module.head_dim <= 256)


def plain_causal(mask: torch.Tensor) -> bool:
    """Whether an attention mask, as attention modules get it (bool or additive
    [batch, 1, tokens, tokens], or [batch, tokens] of the tokens that are there),
    is that of a batch without padding."""
    if mask.dim() == 2:
        return bool((mask != 0).all())
    tokens = mask.shape[-2]
    if mask.shape[-1] != tokens:
        return False
    causal = torch.ones((tokens, tokens), dtype=torch.bool, device=mask.device).tril()
    return bool(((mask if mask.dtype == torch.bool else mask == 0) == causal).all())


class CachedAttention(torch.nn.Module):
    """Wraps an attention module's four projections (the same objects)."""

    def __init__(self, orig_module: torch.nn.Module):
        super().__init__()
        self.training = orig_module.training
        for name in _PARTS:
            setattr(self, name, getattr(orig_module, name))
        # plain attributes callers may read, and the forward for other caches; the
        # module itself is not registered, so parameters keep their names
        for key, val in vars(orig_module).items():
            if not key.startswith("_") and not isinstance(val, torch.nn.Module) and not hasattr(self, key):
                setattr(self, key, val)
        # and share their registry, so that a projection replaced later (quantised,
        # say) is replaced for both
        orig_module.__dict__["_modules"] = self._modules
        self.__dict__["_original"] = orig_module

    def forward(self, hidden_states: torch.Tensor, position_embeddings=None, attention_mask=None,
                past_key_values=None, **kwargs):
        state = getattr(past_key_values, "mi355_cache", None)
        if state is None:
            self._original.training = self.training  # not a registered child: train() and eval() pass it by
            return self._original(hidden_states=hidden_states, position_embeddings=position_embeddings,
                                  attention_mask=attention_mask, past_key_values=past_key_values, **kwargs)
        if attention_mask is not None and not state.unmasked and self.layer_idx == 0 and not plain_causal(attention_mask):
            raise ValueError("the cache's attention takes no mask but a causal one: padding goes behind a row's tokens "
                             "(DecoderCache.new_lens), a draft's tree into DecoderCache.tree_mask")
        batch, tokens, _ = hidden_states.shape
        q, k, v = (proj(hidden_states).view(batch, tokens, -1, self.head_dim)
                   for proj in (self.q_proj, self.k_proj, self.v_proj))
        cache = state.layers[self.layer_idx]
        q = kv_cache_append(cache, k, v, state.lens, new_lens=state.new_lens, q=q, positions=state.positions,
                            inv_freq=state.inv_freq, scale=state.rotary_scale)
        if state.shared_prefix is not None and tokens <= TREE_ATTENTION_MAX_TOKENS:
            out = shared_prefix_attention(q, cache, state.lens, state.shared_prefix, new_lens=state.new_lens,
                                          tree_mask=state.tree_mask, scale=self.scaling)
        elif tokens <= TREE_ATTENTION_MAX_TOKENS:
            out = tree_attention(q, cache, state.lens, new_lens=state.new_lens, tree_mask=state.tree_mask,
                                 scale=self.scaling)
        elif not state.prompt:
            raise ValueError(f"{tokens} tokens behind others: a step takes at most {TREE_ATTENTION_MAX_TOKENS}")
        else:
            if state.tree_mask is not None:
                raise ValueError(f"a tree has at most {TREE_ATTENTION_MAX_TOKENS} tokens, got {tokens}")
            # zeros in the slots of padding, which hold what was there before: causal
            # attention gives them a weight of 0, and 0 times NaN is NaN
            end = state.lens + (tokens if state.new_lens is None else state.new_lens)
            k, v = kv_cache_read(cache, end, tokens, dtype=q.dtype)
            out = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), k, v, is_causal=True,
                                                                   scale=self.scaling, enable_gqa=True).transpose(1, 2)
        return self.o_proj(out.reshape(batch, tokens, -1)), None
