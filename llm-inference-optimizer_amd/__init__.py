"""MI355X-native fused RMSNorm + SwiGLU path for Qwen2-style decoders.

The package directory name contains hyphens, so import it by name with
importlib after putting the repository root on ``sys.path``::

    import importlib, sys
    sys.path.insert(0, "/path/to/repo")
    fk = importlib.import_module("llm-inference-optimizer_amd")
    fk.patch_model_with_fused_kernels(model)

Public surface (the reference's Stage 3 plugin API):

* ``fused_rmsnorm(x, weight, eps=1e-6)``, ``naive_rmsnorm_reference``
* ``fused_silu_mul(gate, up)``, ``naive_silu_mul_reference``
* ``FusedRMSNorm``, ``FusedMLP``, ``patch_model_with_fused_kernels``,
  ``RMSNORM_CLASS_NAMES``, ``MLP_CLASS_NAMES``

and, beyond it, ``fused_add_rmsnorm`` (residual add + RMSNorm in one pass)
with ``FusedDecoderLayer`` / ``DECODER_LAYER_CLASS_NAMES``, which
``patch_model_with_fused_kernels(..., fuse_residual=True)`` installs, and
``GraphedGreedyDecoder``, greedy decoding whose per-token step replays one
captured HIP graph, and ``fused_gate_up_silu`` (gate / up projections +
SiLU-and-mul in one kernel for decode batches), which
``patch_model_with_fused_kernels(..., fuse_gate_up=True)`` lets FusedMLP use,
and ``linear16`` (a 16-bit linear that streams the weights at HBM bandwidth
for decode batches), which ``patch_model_with_fused_kernels(...,
hip_down=True)`` lets FusedMLP use for its down projection.

The reference's weight-only int8 stage sits beside it: ``w8a16_linear`` /
``w8a16_reference``, ``QuantizedLinearInt8`` and ``quantize_model_int8``
(int8 weights with per-output-channel scales, HIP quantiser and W8A16
kernels), composable with the fused-kernel patch.

Between an attention block's projections: ``fused_rotary`` (rotary positions,
``rotary_frequencies`` for long contexts), ``KVCache`` with ``kv_cache_append``,
``kv_cache_read`` and ``kv_cache_keep`` (a paged cache, quantised to int8 or
e4m3 as it is written), and ``tree_attention`` (one new token, or a tree of
drafted ones, over that cache).  ``patch_model_with_fused_kernels(...,
fuse_attention=True)`` installs ``CachedAttention``, with which
``GraphedGreedyDecoder(..., kv_cache="int8")`` decodes over such a cache, and
with ``draft_tokens=n`` verifies drafted trees.

For several continuations of a prompt: ``kv_cache_reserve`` and ``kv_slot_map``
(page tables and slot maps from the requests' lengths),
``shared_prefix_attention`` (a prefix read and computed once for all sequences
that share it) and ``sample_tokens`` (temperature, top-k, top-p and min-p from
given random numbers).  ``GraphedSamplingDecoder`` decodes on them, n samples of
each prompt, the whole step in one graph.

The kernels live in ``libmi355_fused.so`` (gfx950 HIP, C ABI in
``include/mi355_fused.h``), built by ``build.py``.
"""
from .engine.cached_attention import ATTENTION_CLASS_NAMES, CachedAttention, DecoderCache
from .engine.fused_norm_activation_patch import (DECODER_LAYER_CLASS_NAMES, MLP_CLASS_NAMES, RMSNORM_CLASS_NAMES,
                                                 FusedDecoderLayer, FusedMLP, FusedRMSNorm,
                                                 patch_model_with_fused_kernels)
from .engine.graphed_decode import GraphedGreedyDecoder
from .engine.graphed_sampling import GraphedSamplingDecoder
from .kernels.fused_rmsnorm_hip import fused_add_rmsnorm, fused_rmsnorm, naive_rmsnorm_reference
from .kernels.fused_gate_up_hip import GATE_UP_MAX_ROWS, fused_gate_up_silu, naive_gate_up_silu_reference
from .kernels.fused_swiglu_hip import fused_silu_mul, naive_silu_mul_reference
from .kernels.kv_cache_hip import KV_FORMATS, KVCache, kv_cache_append, kv_cache_keep, kv_cache_read
from .kernels.kv_pages_hip import kv_cache_reserve, kv_slot_map
from .kernels.linear16_hip import LINEAR16_MAX_ROWS, linear16
from .kernels.rotary_hip import fused_rotary, rotary_frequencies
from .kernels.sampling_hip import sample_tokens
from .kernels.shared_prefix_hip import shared_prefix_attention
from .kernels.tree_attention_hip import TREE_ATTENTION_MAX_TOKENS, tree_attention
from .kernels.w8a16_matmul_hip import fused_gate_up_silu_w8a16, quantize_int8_weight, w8a16_linear, w8a16_reference
from .quantization.int8 import QuantizedLinearInt8, quantize_model_int8

__all__ = [
    "fused_rmsnorm", "naive_rmsnorm_reference", "fused_silu_mul", "naive_silu_mul_reference",
    "FusedRMSNorm", "FusedMLP", "patch_model_with_fused_kernels", "RMSNORM_CLASS_NAMES", "MLP_CLASS_NAMES",
    "fused_add_rmsnorm", "FusedDecoderLayer", "DECODER_LAYER_CLASS_NAMES", "GraphedGreedyDecoder",
    "fused_gate_up_silu", "naive_gate_up_silu_reference", "GATE_UP_MAX_ROWS",
    "w8a16_linear", "w8a16_reference", "quantize_int8_weight", "QuantizedLinearInt8", "quantize_model_int8",
    "fused_gate_up_silu_w8a16", "linear16", "LINEAR16_MAX_ROWS",
    "fused_rotary", "rotary_frequencies", "KVCache", "KV_FORMATS", "kv_cache_append", "kv_cache_read",
    "kv_cache_keep", "tree_attention", "TREE_ATTENTION_MAX_TOKENS", "CachedAttention", "DecoderCache",
    "ATTENTION_CLASS_NAMES", "kv_cache_reserve", "kv_slot_map", "shared_prefix_attention", "sample_tokens",
    "GraphedSamplingDecoder",
]
