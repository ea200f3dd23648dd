"""Rotary positions on gfx950.

``fused_rotary(x, positions, inv_freq)`` turns the first ``2 * len(inv_freq)``
elements of every head by the angles ``positions * inv_freq`` in one kernel (C
ABI ``mi355_rotary_fwd``), where HF's models build cosine and sine tables in
the model's dtype and apply them with several torch operations.  Angles are
formed and reduced in 64 bits and never rounded to 16, so that far positions
of long contexts keep their precision.

``rotary_frequencies`` gives the frequencies (and the factor on cosine and
sine) of the usual ways to stretch them for long contexts.  The rotation that
a decode step needs is also fused into ``kv_cache_append``.
"""
from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["fused_rotary", "rotary_frequencies"]

# what each rope_type reads
_SCALING_KEYS = {
    "default": set(), "linear": {"factor"}, "ntk": {"factor"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor"},
    "llama3": {"factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"}}


def fused_rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, scale: float = 1.0,
                 interleaved: bool = False) -> torch.Tensor:
    """x: [batch, tokens, heads, head_dim] (fp16, bf16 or fp32; any strides).
    positions: int64 or int32, [batch, tokens] or what broadcasts to it.
    inv_freq: float32 [pairs], 2 * pairs <= head_dim; elements behind the pairs
    are copied.  Pairs are (j, j + pairs), or (2j, 2j + 1) if ``interleaved``;
    cosine and sine are multiplied by ``scale``.  Returns a new contiguous
    tensor of x's shape and dtype (fp32 arithmetic, one rounding).  Inference
    only, as the package's other kernels: no gradient is recorded."""
    return _lib.ext().rotary(x, positions, inv_freq, scale, interleaved)


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """``(inv_freq, scale)`` for ``fused_rotary`` and ``kv_cache_append``:
    ``inv_freq[j] = theta ** (-2j / rotary_dim)``, computed in 64 bits, changed
    for longer contexts by ``scaling`` -- a dict with the keys of HF's
    ``rope_scaling``:

    * ``{"rope_type": "linear", "factor"}``: every frequency / factor.
    * ``{"rope_type": "ntk", "factor"}``: theta * factor ** (d / (d - 2)), which
      leaves the highest frequency and divides the lowest by factor.
    * ``{"rope_type": "yarn", "factor", "original_max_position_embeddings"[,
      "beta_fast" (32), "beta_slow" (1), "attention_factor"]}``: pairs that turn
      more than beta_fast times in the original context keep their frequency,
      those below beta_slow turns take frequency / factor, with a linear ramp
      over the pair index between; scale = attention_factor or
      0.1 ln(factor) + 1.
    * ``{"rope_type": "llama3", "factor", "original_max_position_embeddings",
      "low_freq_factor", "high_freq_factor"}``: the same idea with a ramp over
      the turns themselves, between low_freq_factor and high_freq_factor.

    Other types and keys are refused (None values, "type" beside "rope_type" and
    a "rope_theta" that is theta excepted)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    d, scale = rotary_dim, 1.0
    j = torch.arange(0, d, 2, dtype=torch.float64)
    kind = scaling.get("rope_type", scaling.get("type")) if scaling else "default"
    if kind not in _SCALING_KEYS:
        raise ValueError(f"unknown rope_type {kind!r} ({', '.join(_SCALING_KEYS)})")
    unknown = {k for k, v in (scaling or {}).items() if v is not None and not (k == "rope_theta" and v == theta)}
    unknown -= _SCALING_KEYS[kind] | {"rope_type", "type"}
    if unknown:
        raise ValueError(f"rope_type {kind!r} does not take {', '.join(sorted(unknown))}")
    if kind == "ntk":
        theta = theta * scaling["factor"] ** (d / (d - 2)) if d > 2 else theta
    freq = theta ** (-j / d)
    if kind == "linear":
        freq = freq / scaling["factor"]
    elif kind == "yarn":
        factor, context = scaling["factor"], scaling["original_max_position_embeddings"]

        def pair_of(turns):  # the (real) pair index that makes so many turns in the original context
            return d * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low = max(math.floor(pair_of(scaling.get("beta_fast") or 32)), 0)
        high = min(math.ceil(pair_of(scaling.get("beta_slow") or 1)), d - 1)
        ramp = ((j / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        scale = scaling.get("attention_factor") or (0.1 * math.log(factor) + 1 if factor > 1 else 1.0)
    elif kind == "llama3":
        turns = scaling["original_max_position_embeddings"] * freq / (2 * math.pi)
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / scaling["factor"] * (1 - keep)
    return freq.to(device=device, dtype=torch.float32), float(scale)
