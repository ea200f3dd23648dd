"""Drawing the next tokens from logits with temperature, top-k, top-p and min-p, on gfx950.  C ABI
``mi355_sample_tokens_fwd``.  The reference's engines only take the argmax (src/engine/graphed_decode_engine.py:141).
"""
from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["sample_tokens"]


def _setting(name: str, value, low: float, high: float):
    """(tensor, 0) or (None, number) of a setting that is per row or for all."""
    if torch.is_tensor(value):
        return value, 0
    if not (isinstance(value, (int, float)) and low <= value <= high):  # NaN is refused too
        raise ValueError(f"{name} must be a tensor or a number in [{low:g}, {high:g}], got {value!r}")
    return None, value


def sampling_settings(temperature, top_k, top_p, min_p):
    """The four as ``_setting`` has them; ValueError for a number that ``sample_tokens`` does not take."""
    heat = _setting("temperature", temperature, 0.0, math.inf)
    k = _setting("top_k", top_k, 0, 2 ** 31 - 1)
    if int(k[1]) != k[1]:
        raise ValueError(f"top_k must be a whole number, got {top_k!r}")
    return heat, k, _setting("top_p", top_p, 0.0, 1.0), _setting("min_p", min_p, 0.0, 1.0)


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
                  return_logprobs: bool = False):
    """One token per row of ``logits`` [..., vocab] (fp16, bf16 or fp32; rows of any stride): int64 [...]; with
    ``return_logprobs`` also the logarithm of the probability that it was drawn with, float32 [...].

    Rows are drawn with the given numbers ``uniform`` (float32 [...], in [0, 1), ``torch.rand``'s, say), so the same
    numbers give the same tokens.  Each setting is a number, or a tensor [...] with one for each row (float32; top_k
    int32).  Of a row's tokens, ranked by their logit (equal ones by index), those stay that

    * are among the first ``top_k`` (0: all),
    * of these, are the fewest that have at least ``top_p`` of the probability (1: all), and
    * have at least ``min_p`` times the probability of the most probable one (0: all),

    with probabilities after dividing the logits by ``temperature``; the token is the first, in the order of the
    vocabulary, at which their cumulated probability exceeds ``uniform``.  A temperature of 0 takes the first of the
    largest logits.  Probabilities and their sums are held in 64 bits.  -infinity and NaN are never drawn; a row of
    nothing else gets -1 (and a logarithm of -infinity).

    Rows of 151936 take 30 to 90 us, but about a millisecond where the last token that ``top_k`` keeps has less than
    2^-63 of the largest's probability (low temperatures, masks that leave fewer tokens), or a limit of many tokens
    falls into a flat part of the row (high temperatures, a ``top_p`` near 1)."""
    (heat, heat_all), (k, k_all), (p, p_all), (least, least_all) = sampling_settings(temperature, top_k, top_p, min_p)
    tokens, logs = _lib.ext().sample(logits, uniform, heat, heat_all, k, int(k_all), p, p_all, least, least_all,
                                     return_logprobs)
    return (tokens, logs) if return_logprobs else tokens
