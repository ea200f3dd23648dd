"""Greedy decoding whose per-token step replays one captured HIP graph.

The caller the reference's Stage 6 engine provides
(src/engine/graphed_decode_engine.py:47-186, GraphedDecodeEngine), rebuilt on
HF's own ``StaticCache`` instead of the reference's paged KV cache (paged
attention is not on this path): every buffer the decode step touches is
allocated once, the step reads only static tensors (the current tokens and
the cache position), and after the first step the whole forward pass -- 28
layers of attention, the fused RMSNorm / SiLU-and-mul kernels, GEMMs and LM
head -- is one graph replay.  As in the reference (:129-147), the graph
is replayed right after capture, so the first captured step also returns a
computed result rather than whatever the capture pass left behind.  The argmax
stays outside: over a vocabulary torch splits it over workgroups that count
themselves in memory which a memset clears before, and a memset replayed as a
graph node may not have cleared it -- then nobody writes the result.

It works with the patched and the unpatched model alike; the fused kernels
enqueue no allocation, sync or memset, so they capture cleanly.

With ``kv_cache="int8"`` (or "e4m3", "16bit") the step's keys and values go to
a paged cache of that format instead of HF's StaticCache, and attention runs on
this package's kernels over the tokens there are instead of the whole buffer
(engine/cached_attention.py).  With ``draft_tokens=n`` on top, every step
verifies a tree of up to n drafted tokens per sequence (engine/
prompt_lookup.py) and keeps the longest branch that greedy decoding agrees
with: fewer, somewhat larger steps for the same tokens.
"""
from __future__ import annotations

import torch

from ..kernels.tree_attention_hip import TREE_ATTENTION_MAX_TOKENS
from .cached_attention import DecoderCache
from .prompt_lookup import TextIndex, accept, draft_tree

__all__ = ["GraphedGreedyDecoder"]


class GraphedGreedyDecoder:
    """Greedy generation for an HF causal LM with a graph-captured decode step.

    ``batch_size`` and ``max_cache_len`` fix the static buffers (one graph per
    decoder).  ``generate(input_ids, max_new_tokens)`` returns the prompt
    followed by the generated tokens, like ``generate_graphed`` in the
    reference (:177-186); with ``return_logits=True`` it also returns the
    last-position logits behind each generated token, [batch, new, vocab]
    (the prefill's, then each step's).  ``use_graph=False`` runs the
    identical static-cache step eagerly (for comparison).

    ``kv_cache``: "int8", "e4m3" or "16bit" keeps keys and values in a
    ``KVCache`` of that format (pages of ``page_size`` slots, a multiple of 16;
    one page per sequence without it).  The model's attention has to be patched
    (``patch_model_with_fused_kernels(model, fuse_attention=True)``).
    ``draft_tokens`` (2 .. 128, only with ``kv_cache``): nodes of the tree that a
    step verifies; ``steps`` counts the steps of the last generation.  They pay
    for single sequences that repeat themselves; a batch takes the steps of its
    slowest sequence, each with host work per sequence, and may get slower.  Tokens are
    those of greedy decoding up to rounding: a step of several tokens runs its
    projections in other shapes, so that near-ties may fall the other way."""

    def __init__(self, model, batch_size: int, max_cache_len: int, use_graph: bool = True,
                 kv_cache: str | None = None, page_size: int | None = None, draft_tokens: int | None = None):
        self.model = model
        self.device = next(model.parameters()).device
        self.batch_size = batch_size
        self.max_cache_len = max_cache_len
        self.use_graph = use_graph
        self.draft_tokens = draft_tokens
        self.steps = 0
        if kv_cache is None and (draft_tokens is not None or page_size is not None):
            raise ValueError("draft_tokens and page_size need kv_cache")
        if draft_tokens is not None and not 2 <= draft_tokens <= TREE_ATTENTION_MAX_TOKENS:
            raise ValueError(f"draft_tokens must be in [2, {TREE_ATTENTION_MAX_TOKENS}], got {draft_tokens}")
        if kv_cache is not None:
            self._init_cached(kv_cache, page_size)
            return
        from transformers import StaticCache

        self.cache = StaticCache(config=model.config, max_cache_len=max_cache_len)
        self._tok = torch.zeros((batch_size, 1), dtype=torch.long, device=self.device)
        self._pos = torch.zeros((1,), dtype=torch.long, device=self.device)
        self._pos0 = self._pos.view(())  # 0-d view for the cache's write counters
        self._pos_ids = torch.zeros((batch_size, 1), dtype=torch.long, device=self.device)
        self._logits = None
        self._graph = None

    def _init_cached(self, kv_cache: str, page_size: int | None) -> None:
        n, t = self.batch_size, self.draft_tokens or 1
        # a draft's last nodes may lie behind the last token that is wanted
        self.cache = DecoderCache.allocate(self.model, n, self.max_cache_len + t - 1, kv_cache, page_size)
        self.cache.unmasked = True
        self._past = self.cache.as_past()
        self._tok = torch.zeros((n, t), dtype=torch.long, device=self.device)
        self._pos_ids = torch.zeros((n, t), dtype=torch.long, device=self.device)
        if self.draft_tokens:
            self._new_lens = torch.zeros((n,), dtype=torch.int32, device=self.device)
            self._mask = torch.zeros((n, t, t), dtype=torch.bool, device=self.device)
            self._kept = torch.zeros((n, t), dtype=torch.int32, device=self.device)
            self._kept_lens = torch.zeros((n,), dtype=torch.int32, device=self.device)
        self._logits = None
        self._graph = None

    def _cached_forward(self, ids: torch.Tensor, positions: torch.Tensor, new_lens=None, tree_mask=None, prompt=False):
        c = self.cache
        c.positions, c.new_lens, c.tree_mask, c.prompt = positions, new_lens, tree_mask, prompt
        out = self.model(input_ids=ids, past_key_values=self._past, position_ids=positions, use_cache=True,
                         logits_to_keep=1 if prompt else 0)
        return out.logits

    def _cached_step(self) -> torch.Tensor:
        """One token per sequence, or a draft: first the last draft's accepted
        tokens move together and become part of the cache."""
        if not self.draft_tokens:
            logits = self._cached_forward(self._tok, self._pos_ids)[:, -1]
            self.cache.lens.add_(1)
            return logits
        self.cache.keep(self._kept, self._kept_lens)
        self.cache.lens.add_(self._kept_lens)
        return self._cached_forward(self._tok, self._pos_ids, self._new_lens, self._mask)

    def _step_logits(self) -> torch.Tensor:
        """What the graph holds."""
        if isinstance(self.cache, DecoderCache):
            return self._cached_step()
        # HF's StaticLayer writes at its own device-side counter
        # (cumulative_length) and bumps it in place; pin every layer's counter
        # to the cache position first, so warm-up, capture and replays all
        # write the token at its position (one multi-tensor copy kernel).
        counters = [layer.cumulative_length for layer in self.cache.layers]
        torch._foreach_copy_(counters, [self._pos0] * len(counters))
        out = self.model(input_ids=self._tok, past_key_values=self.cache, cache_position=self._pos,
                         position_ids=self._pos_ids, use_cache=True)
        return out.logits[:, -1]

    def _picks(self, logits: torch.Tensor) -> torch.Tensor:
        return logits.argmax(-1, keepdim=not self.draft_tokens)

    def _step(self) -> tuple[torch.Tensor, torch.Tensor]:
        logits = self._step_logits()
        return logits, self._picks(logits)

    def _capture(self) -> None:
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        cached = isinstance(self.cache, DecoderCache)
        if cached:  # the warm-up step moves the cache on, and is taken back: the captured step writes the same slots
            lens = self.cache.lens.clone()
            side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            self._step_logits()  # warm-up: kernel selection and lazy allocations happen outside the capture
        torch.cuda.current_stream(self.device).wait_stream(side)
        if cached:
            self.cache.lens.copy_(lens)
        torch.cuda.synchronize(self.device)
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self._logits = self._step_logits()

    def _run(self) -> tuple[torch.Tensor, torch.Tensor]:
        """One step, replayed (captured at first) or eager; the graph's logits
        are overwritten by the next."""
        self.steps += 1
        if not self.use_graph:
            return self._step()
        if self._graph is None:
            self._capture()
        self._graph.replay()
        return self._logits, self._picks(self._logits)

    def _cached_prompt(self, input_ids: torch.Tensor) -> torch.Tensor:
        """The prompt into an empty cache; its last logits."""
        B, S = input_ids.shape
        self.cache.lens.zero_()
        pos = torch.arange(S, device=self.device).unsqueeze(0).expand(B, S)
        logits = self._cached_forward(input_ids, pos, prompt=True)[:, -1]
        self.cache.lens.fill_(S)
        return logits

    def _generate_drafted(self, input_ids: torch.Tensor, max_new_tokens: int, return_logits: bool):
        B, S = input_ids.shape
        t = self.draft_tokens
        logits = self._cached_prompt(input_ids)
        seqs = [TextIndex(row) for row in input_ids.tolist()]
        for s, tok in zip(seqs, logits.argmax(-1).tolist()):
            s.extend([tok])
        done = S + max_new_tokens
        kept_logits = [[row.to(torch.float32, copy=True)] for row in logits] if return_logits else None
        self._kept_lens.zero_()
        while any(len(s) < done for s in seqs):
            trees = [draft_tree(s, t) if len(s) < done else ([], []) for s in seqs]
            tok, pos = [[0] * t for _ in seqs], [[0] * t for _ in seqs]
            mask = [[[False] * t for _ in range(t)] for _ in seqs]
            for b, (nodes, parents) in enumerate(trees):
                tok[b][:len(nodes)] = nodes
                for i, parent in enumerate(parents):
                    if i:
                        mask[b][i] = list(mask[b][parent])
                    mask[b][i][i] = True
                    pos[b][i] = len(seqs[b]) - 1 if i == 0 else pos[b][parent] + 1
            self._tok.copy_(torch.tensor(tok))
            self._pos_ids.copy_(torch.tensor(pos))
            self._mask.copy_(torch.tensor(mask))
            self._new_lens.copy_(torch.tensor([len(n) for n, _ in trees], dtype=torch.int32))
            logits, picks = self._run()
            picks = picks.tolist()
            kept, counts = torch.zeros((B, t), dtype=torch.int32), torch.zeros((B,), dtype=torch.int32)
            for b, (nodes, parents) in enumerate(trees):
                if not nodes:
                    continue
                path = accept(nodes, parents, picks[b])[:done - len(seqs[b])]
                kept[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
                counts[b] = len(path)
                seqs[b].extend([picks[b][i] for i in path])
                if return_logits:
                    kept_logits[b] += [logits[b, i].to(torch.float32, copy=True) for i in path]
            self._kept.copy_(kept)
            self._kept_lens.copy_(counts)
        # the last step's accepted tokens, as the next step would move them
        self.cache.keep(self._kept, self._kept_lens)
        self.cache.lens.add_(self._kept_lens)
        self._kept_lens.zero_()
        ids = torch.tensor([s.tokens for s in seqs], dtype=torch.long, device=self.device)
        return (ids, torch.stack([torch.stack(r) for r in kept_logits])) if return_logits else ids

    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, return_logits: bool = False):
        B, S = input_ids.shape
        if B != self.batch_size:
            raise ValueError(f"batch size {B} != the decoder's {self.batch_size}")
        if S + max_new_tokens > self.max_cache_len:
            raise ValueError(f"{S} + {max_new_tokens} tokens exceed max_cache_len {self.max_cache_len}")
        self.steps = 0
        cached = isinstance(self.cache, DecoderCache)
        if self.draft_tokens:
            return self._generate_drafted(input_ids, max_new_tokens, return_logits)
        if cached:
            logits = self._cached_prompt(input_ids)
        else:
            self.cache.reset()
            pos = torch.arange(S, device=self.device)
            out = self.model(input_ids=input_ids, past_key_values=self.cache, cache_position=pos,
                             position_ids=pos.unsqueeze(0).expand(B, S), use_cache=True)
            logits = out.logits[:, -1]
        tok = logits.argmax(-1, keepdim=True)
        toks = [tok]
        step_logits = [logits.to(torch.float32, copy=True)] if return_logits else None
        for i in range(max_new_tokens - 1):
            self._tok.copy_(tok)
            if not cached:
                self._pos.fill_(S + i)
            self._pos_ids.fill_(S + i)
            logits, tok = self._run()
            toks.append(tok)
            if return_logits:
                # a copy: the graph's output buffer is rewritten by the next replay
                step_logits.append(logits.to(torch.float32, copy=True))
        ids = torch.cat([input_ids] + toks, dim=1)
        return (ids, torch.stack(step_logits, dim=1)) if return_logits else ids
