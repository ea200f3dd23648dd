"""Several sampled continuations of each prompt, whose per-token step replays one captured HIP graph.

``GraphedSamplingDecoder`` keeps every prompt's keys and values once.  Its step

    kv_cache_reserve (a page for the sequences that enter a new one) -> forward, in every layer kv_cache_append and
    shared_prefix_attention (the prompt read and computed once for all of its continuations; of short ones
    tree_attention) -> sample_tokens

reads and writes static tensors only, so that all of it is one graph: the page table grows, tokens are drawn and fed
back on the GPU, and the host adds a step's random numbers.  (The greedy decoder's argmax has to stay outside; the
package's kernels leave nothing for a memset to clear.)

The reference's engines decode greedily, one continuation per prompt (src/engine/graphed_decode_engine.py:47-186).
"""
from __future__ import annotations

import torch

from ..kernels.kv_cache_hip import KVCache
from ..kernels.kv_pages_hip import kv_cache_reserve, kv_slot_map
from ..kernels.sampling_hip import sample_tokens, sampling_settings
from .cached_attention import DecoderCache

__all__ = ["GraphedSamplingDecoder"]

# What a layer's tree_attention has to read of the prompts, each once per continuation, from which on
# shared_prefix_attention is the faster: it has two kinds of pieces to start and to join.  In a graph, int8, 128-wide
# heads, us of shared_prefix_attention and tree_attention: 12 / 2 heads, 1 x 8 continuations of 1024 tokens (4 MB) 16.1
# and 10.5; 1 x 32 of 4096 (69 MB) 24.9 and 23.3; 4 x 8 of 4096 (69) 23.2 and 24.7; 4 x 16 of 8192 (277) 32.4 and 60.5;
# 28 / 4 heads, 4 x 8 of 1024 (35) 22.4 and 19.9; of 2048 (69) 24.4 and 26.7.
_SHARED_BYTES = 64 << 20


class GraphedSamplingDecoder:
    """Sampled generation for an HF causal LM whose attention is patched (``patch_model_with_fused_kernels(model,
    fuse_attention=True)``): ``samples`` continuations of each of ``batch_size`` prompts.

    ``kv_cache``: "16bit", "int8" or "e4m3", in pages of ``page_size`` slots.  ``pages``: how many the pool holds; a
    generation of ``new`` tokens takes ``pages_needed(prompt length, new)`` of them, far fewer than the default, which
    is enough for sequences of ``max_cache_len`` tokens that share nothing.  ``temperature``, ``top_k``, ``top_p`` and
    ``min_p`` as in ``sample_tokens``: numbers, or tensors that broadcast to [batch_size, samples], which are copied.
    ``share_prefix``: whether attention reads a prompt once for all of its continuations (``shared_prefix_attention``)
    or for each (``tree_attention``); None: whichever is faster at the prompt's length.  ``use_graph=False`` runs the
    same step eagerly."""

    def __init__(self, model, batch_size: int, samples: int, max_cache_len: int, *, kv_cache: str = "16bit",
                 page_size: int = 64, pages: int | None = None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 share_prefix: bool | None = None, use_graph: bool = True):
        if batch_size < 1 or samples < 1:
            raise ValueError(f"batch_size and samples must be at least 1, got {batch_size} and {samples}")
        sampling_settings(temperature, top_k, top_p, min_p)
        self.model = model
        self.device = next(model.parameters()).device
        self.batch_size, self.samples, self.max_cache_len = batch_size, samples, max_cache_len
        self.page_size, self.share_prefix, self.use_graph = page_size, share_prefix, use_graph
        rows = batch_size * samples
        self.pages = rows * -(-max_cache_len // page_size) if pages is None else pages
        self.settings = {name: self._per_row(value, torch.int32 if name == "top_k" else torch.float32)
                         for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p),
                                             ("min_p", min_p))}
        self.cache = DecoderCache.allocate(model, rows, max_cache_len, kv_cache, page_size, self.pages)
        self.cache.unmasked = True
        self.table = self.cache.layers[0].page_table
        # the prompts, in the first row of each: the same pools through every `samples`-th row of the table
        self.prompt_cache = DecoderCache([KVCache(c.k, c.v, self.table[::samples], c.k_scale, c.v_scale)
                                          for c in self.cache.layers], self.cache.inv_freq, self.cache.rotary_scale)
        self.prompt_cache.unmasked = self.prompt_cache.prompt = True
        self._prefix = torch.zeros((batch_size,), dtype=torch.int32, device=self.device)
        self._past, self._prompt_past = self.cache.as_past(), self.prompt_cache.as_past()
        self._one = torch.ones((rows,), dtype=torch.int32, device=self.device)
        self._missing = torch.zeros((rows,), dtype=torch.int32, device=self.device)
        self._drawn = torch.zeros((rows,), dtype=torch.long, device=self.device)  # below 0: a draw gave no token
        self._tok = torch.zeros((rows, 1), dtype=torch.long, device=self.device)
        self._pos = torch.zeros((rows, 1), dtype=torch.long, device=self.device)
        self._uniform = torch.zeros((rows,), dtype=torch.float32, device=self.device)
        self._log = torch.zeros((rows,), dtype=torch.float32, device=self.device)
        self._graph, self._graphs = None, {}

    def _per_row(self, value, dtype):
        if not torch.is_tensor(value):
            return value
        own = torch.empty((self.batch_size, self.samples), dtype=dtype, device=self.device)
        if dtype == torch.int32 and value.dtype == torch.int64:  # in 32 bits 2^32 + 1 would be another limit
            value = value.clamp(0, 2 ** 31 - 1)
        return own.copy_(value.detach().expand_as(own)).view(-1)

    def pages_needed(self, prompt_len: int, new_tokens: int) -> int:
        """Pages of a generation: the prompts', and what each continuation has for itself."""
        shared = prompt_len // self.page_size
        end = -(-(prompt_len + new_tokens - 1) // self.page_size)
        return self.batch_size * (shared + self.samples * (end - shared))

    def _shares(self, length: int) -> bool:
        if self.share_prefix is not None:
            return self.share_prefix
        c = self.cache.layers[0]
        token = 2 * c.k.shape[1] * (c.k.shape[3] * c.k.element_size() + (4 if c.k_scale is not None else 0))
        return self.samples > 1 and self.batch_size * self.samples * length * token >= _SHARED_BYTES

    def _sample(self, logits: torch.Tensor) -> None:
        """Draws the rows' next tokens into the step's inputs."""
        tokens, logs = sample_tokens(logits, self._uniform, return_logprobs=True, **self.settings)
        torch.minimum(self._drawn, tokens, out=self._drawn)  # -1 where all logits are NaN: generate tells it
        self._tok.copy_(tokens.clamp_(min=0).unsqueeze(1))
        self._log.copy_(logs)

    def _step(self) -> None:
        c = self.cache
        self._missing.copy_(torch.maximum(self._missing, kv_cache_reserve(c.layers[0], c.lens, self._one)[1]))
        c.positions = self._pos
        out = self.model(input_ids=self._tok, past_key_values=self._past, position_ids=self._pos, use_cache=True)
        c.lens.add_(1)
        self._pos.add_(1)
        self._sample(out.logits[:, -1])

    def _capture(self) -> None:
        state = (self.cache.lens, self._pos, self._tok, self._log, self._missing, self._drawn, self.table)
        held = [t.clone() for t in state]
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            self._step()  # warm-up, taken back below: the captured step writes the same slots
        torch.cuda.current_stream(self.device).wait_stream(side)
        for t, old in zip(state, held):
            t.copy_(old)
        torch.cuda.synchronize(self.device)
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self._step()

    def _prompts(self, input_ids: torch.Tensor) -> torch.Tensor:
        """The prompts into an empty cache, each once; every continuation's table names their whole pages and a page of
        its own with a copy of the rest.  Their last logits."""
        (n, length), m, page, c = input_ids.shape, self.samples, self.page_size, self.cache
        self.table.fill_(-1)
        c.lens.zero_()
        self._missing.zero_()
        self._drawn.zero_()
        new = torch.zeros((n, m), dtype=torch.int32, device=self.device)
        new[:, 0] = length
        kv_cache_reserve(c.layers[0], c.lens, new.view(-1))
        p = self.prompt_cache
        p.lens.zero_()
        p.positions = torch.arange(length, device=self.device).unsqueeze(0).expand(n, length)
        logits = self.model(input_ids=input_ids, past_key_values=self._prompt_past, position_ids=p.positions,
                            use_cache=True, logits_to_keep=1).logits[:, -1]
        shared = length // page
        rows = self.table.view(n, m, -1)
        rows[:, 1:, :shared] = rows[:, :1, :shared]
        c.lens.fill_(length)
        kv_cache_reserve(c.layers[0], c.lens)
        rest = length - shared * page
        if rest and m > 1:
            slots = kv_slot_map(c.layers[0], torch.full_like(c.lens, shared * page), torch.full_like(c.lens, rest),
                                n * m * rest)[0].view(n, m, rest)
            to, source = slots[:, 1:], slots[:, :1].expand(n, m - 1, rest)
            for layer in c.layers:
                for t in (layer.k, layer.v, layer.k_scale, layer.v_scale):
                    if t is not None:
                        t = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
                        t[to // page, :, to % page] = t[source // page, :, source % page]
        self._prefix.fill_(shared * page)
        shares = self._shares(length)
        c.shared_prefix = self._prefix if shares else None
        self._graph = self._graphs.get(shares)
        self._pos.fill_(length)
        return logits

    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, uniform: torch.Tensor | None = None,
                 generator: torch.Generator | None = None, return_logprobs: bool = False):
        """input_ids [batch_size, length] -> [batch_size, samples, length + max_new_tokens]; with ``return_logprobs``
        also the logarithm of the probability that each new token was drawn with.  ``uniform``: the random numbers
        (float32 [batch_size, samples, max_new_tokens]); without it ``torch.rand``'s, from ``generator``.  RuntimeError
        if a row's logits were all NaN or -infinity, so that there was no token to draw."""
        n, length = input_ids.shape
        m, rows = self.samples, self.batch_size * self.samples
        if n != self.batch_size:
            raise ValueError(f"batch size {n} != the decoder's {self.batch_size}")
        if max_new_tokens < 1 or length < 1 or length + max_new_tokens > self.max_cache_len:
            raise ValueError(f"{length} + {max_new_tokens} tokens: both at least 1, at most {self.max_cache_len} together")
        if self.pages_needed(length, max_new_tokens) > self.pages:
            raise ValueError(f"{length} + {max_new_tokens} tokens take {self.pages_needed(length, max_new_tokens)} pages, "
                             f"the pool has {self.pages}")
        shape = (n, m, max_new_tokens)
        if uniform is None:
            uniform = torch.rand(shape, generator=generator, device=self.device if generator is None else generator.device)
        if uniform.shape != shape:
            raise ValueError(f"uniform must be {shape}, got {tuple(uniform.shape)}")
        uniform = uniform.to(device=self.device, dtype=torch.float32).reshape(rows, max_new_tokens)
        out = torch.empty((rows, max_new_tokens), dtype=torch.long, device=self.device)
        logs = torch.empty((rows, max_new_tokens), dtype=torch.float32, device=self.device)
        logits = self._prompts(input_ids)
        self._uniform.copy_(uniform[:, 0])
        self._sample(logits.unsqueeze(1).expand(n, m, -1).reshape(rows, -1))
        for i in range(max_new_tokens):
            if i:
                self._uniform.copy_(uniform[:, i])
                if not self.use_graph:
                    self._step()
                else:
                    if self._graph is None:
                        self._capture()
                        self._graphs[self.cache.shared_prefix is not None] = self._graph
                    self._graph.replay()
            out[:, i] = self._tok[:, 0]
            logs[:, i] = self._log
        if bool((self._missing > 0).any()):
            raise RuntimeError("the cache's pool ran out of pages")
        if bool((self._drawn < 0).any()):
            raise RuntimeError("a row's logits left no token to draw: they were all NaN or -infinity")
        ids = torch.cat((input_ids.unsqueeze(1).expand(n, m, length), out.view(shape)), 2)
        return (ids, logs.view(shape)) if return_logprobs else ids
