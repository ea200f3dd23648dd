"""GraphedGreedyDecoder over the quantised cache, with and without drafted trees, against an independent prefill of
the decoded sequence into HF's DynamicCache: what the cache holds, the logits behind every token, and the tokens."""
import pytest
import torch

from decode_check import compare_logits, reference_pass, sharpen_attention

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")

LAYERS, VOCAB = 4, 512
# What 8 bits in every key and value do to 4 layers: a step is at most 1/127 (int8: half of it off, 0.4% of a row's
# largest) or 1/16 (e4m3: half of that, 3% of the value) -- in the attention's output, through the rest of the layers,
# no more than that again per layer on values of order one.  A slot written to the wrong place is off by order one.
CACHE_TOL = {"16bit": 0.03, "int8": 0.06, "e4m3": 0.3}
LOGIT_TOL = {"16bit": 0.05, "int8": 0.2, "e4m3": 1.0}  # on logits of about 4


def _model(cuda, heads=4, kv_heads=2, hidden=256, seed=3, dtype=torch.float16, vocab=VOCAB, **kw):
    cfg = transformers.Qwen2Config(vocab_size=vocab, hidden_size=hidden, intermediate_size=512,
                                   num_hidden_layers=LAYERS, num_attention_heads=heads, num_key_value_heads=kv_heads,
                                   max_position_embeddings=4096, rms_norm_eps=1e-6, tie_word_embeddings=True,
                                   attn_implementation="sdpa", initializer_range=0.06,
                                   rope_parameters={"rope_theta": 1e6, "rope_type": "default"}, **kw)
    torch.manual_seed(seed)
    with torch.device(cuda):
        m = transformers.Qwen2ForCausalLM(cfg)
    m = m.to(dtype).eval()
    sharpen_attention(m, 1.5)
    return m


def _prompt(cuda, batch, length, seed=11, period=None):
    ids = torch.randint(0, VOCAB, (batch, period or length), generator=torch.Generator().manual_seed(seed))
    return ids.repeat(1, -(-length // ids.shape[1]))[:, :length].to(cuda)


def _check(pkg, model, dec, ids, out, logits, kind, what):
    n = ids.shape[1]
    new = out[:, n:]
    assert torch.equal(out[:, :n], ids) and torch.equal(logits.argmax(-1), new)
    ref_logits, ref_cache = reference_pass(model, ids, new)
    r = compare_logits(new, logits, ref_logits)
    held = out.shape[1] - 1
    assert dec.cache.lens.tolist() == [held] * out.shape[0]
    worst = 0.0
    for cache, ref in zip(dec.cache.layers, ref_cache.layers):
        k, v = pkg.kv_cache_read(cache, dec.cache.lens, held, dtype=ref.keys.dtype)
        for got, want in ((k, ref.keys), (v, ref.values)):
            per_slot = (got.float() - want.float()).abs().amax((0, 1, 3)) / want.float().abs().max()
            worst = max(worst, per_slot.max().item())
    print(f"{what}: steps {dec.steps}, cache off by {worst:.3g}, logits by {r['noise']:.3g} of {r['logit_scale']:.3g}, "
          f"{r['mismatch_frac']:.2%} other picks (gap {r['max_gap_at_mismatch']:.3g})")
    assert worst <= CACHE_TOL[kind]
    assert r["noise"] <= LOGIT_TOL[kind]
    assert r["max_gap_at_mismatch"] <= 2 * r["noise"] + 1e-6


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("length", [9, 200])  # below and beyond what tree_attention takes at once
def test_decode_over_the_cache(pkg, cuda, kind, length):
    model = _model(cuda)
    assert pkg.patch_model_with_fused_kernels(model, fuse_attention=True, fuse_residual=True)["attention"] == LAYERS
    ids = _prompt(cuda, 3, length)
    dec = pkg.GraphedGreedyDecoder(model, 3, 300, kv_cache=kind, page_size=32)
    out, logits = dec.generate(ids, 30, return_logits=True)
    assert dec._graph is not None and dec.steps == 29
    _check(pkg, model, dec, ids, out, logits, kind, f"{kind} {length}")
    # the same steps without a graph, then another prompt through the captured graph
    eager = pkg.GraphedGreedyDecoder(model, 3, 300, use_graph=False, kv_cache=kind, page_size=32)
    assert all(torch.equal(a, b) for a, b in zip(eager.generate(ids, 30, return_logits=True), (out, logits)))
    ids2 = _prompt(cuda, 3, 17, seed=12)
    graph = dec._graph
    out2, logits2 = dec.generate(ids2, 20, return_logits=True)
    assert dec._graph is graph
    _check(pkg, model, dec, ids2, out2, logits2, kind, f"{kind} again")


@pytest.mark.parametrize("kind", ["16bit", "int8"])
@pytest.mark.parametrize("draft,use_graph", [(2, True), (12, True), (12, False), (40, True)])
def test_decode_with_drafts(pkg, cuda, kind, draft, use_graph):
    """Prompts that repeat themselves, so that drafts are found; every token is still checked against the
    independent pass, and the cache holds the accepted tokens alone, in order."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    dec = pkg.GraphedGreedyDecoder(model, 3, 200, use_graph=use_graph, kv_cache=kind, draft_tokens=draft)
    ids = torch.cat((_prompt(cuda, 2, 40, period=7), _prompt(cuda, 1, 40, seed=13)))
    for new in (60, 1, 2):
        out, logits = dec.generate(ids, new, return_logits=True)
        assert out.shape == (3, 40 + new) and logits.shape == (3, new, VOCAB) and dec.steps <= max(0, new - 1)
        _check(pkg, model, dec, ids, out, logits, kind, f"{kind} draft {draft} new {new}")


@pytest.mark.parametrize("draft", [5, 24])
def test_drafts_that_are_accepted(pkg, cuda, draft):
    """A vocabulary of 8: the text repeats its n-grams, and steps accept several tokens, other branches than the first
    among them."""
    model = _model(cuda, vocab=8)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = _prompt(cuda, 4, 30) % 8
    dec = pkg.GraphedGreedyDecoder(model, 4, 200, kv_cache="16bit", draft_tokens=draft)
    out, logits = dec.generate(ids, 150, return_logits=True)
    _check(pkg, model, dec, ids, out, logits, "16bit", f"draft {draft}")
    assert dec.steps < 149


@pytest.mark.parametrize("kv,draft", [(None, None), ("16bit", None), ("int8", None), ("int8", 6)])
def test_a_large_vocabulary(pkg, cuda, kv, draft):
    """Many replays with a vocabulary over which an argmax takes more than one workgroup, and eager work between."""
    model = _model(cuda, vocab=151936)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=kv is not None)
    dec = pkg.GraphedGreedyDecoder(model, 1, 160, **({} if kv is None else dict(kv_cache=kv, draft_tokens=draft)))
    for seed in (1, 2, 3):
        ids = _prompt(cuda, 1, 50, seed=seed)
        out, logits = dec.generate(ids, 40, return_logits=True)
        assert torch.equal(logits.argmax(-1), out[:, 50:]) and out.min() >= 0 and out.max() < 151936
        again = dec.generate(ids, 40)
        assert torch.equal(again, out)


def test_bf16_wide_heads_and_int8_weights(pkg, cuda):
    """Heads of 128, bf16, weights quantised after the patch (the attention's projections among them)."""
    model = _model(cuda, heads=4, kv_heads=1, hidden=512, dtype=torch.bfloat16)
    counts = pkg.patch_model_with_fused_kernels(model, fuse_attention=True, fuse_gate_up=True, hip_down=True)
    assert counts["attention"] == LAYERS
    assert pkg.quantize_model_int8(model)["layers_quantized"] == 7 * LAYERS
    block = model.model.layers[0].self_attn
    assert isinstance(block.q_proj, pkg.QuantizedLinearInt8) and block._original.q_proj is block.q_proj
    ids = _prompt(cuda, 2, 33)
    dec = pkg.GraphedGreedyDecoder(model, 2, 100, kv_cache="16bit")
    out, logits = dec.generate(ids, 20, return_logits=True)
    assert torch.equal(logits.argmax(-1), out[:, 33:])
    ref_logits, _ = reference_pass(model, ids, out[:, 33:])
    # bf16 has 3 bits fewer than fp16, and logits, sums over the hidden elements, grow with sqrt(512 / 256): 8 sqrt 2
    assert (logits - ref_logits).abs().max().item() <= 8 * 2 ** 0.5 * LOGIT_TOL["16bit"]


def test_other_caches_are_unchanged(pkg, cuda):
    """A patched model with HF's own caches computes what it did, bit for bit."""
    model, ids = _model(cuda), _prompt(cuda, 2, 30)
    with torch.inference_mode():
        want = model(ids).logits
        names = [n for n, _ in model.named_parameters()]
        pkg.patch_model_with_fused_kernels(model, patch_norm=False, patch_mlp=False, fuse_attention=True)
        assert torch.equal(model(ids).logits, want)
    assert [n for n, _ in model.named_parameters()] == names
    a = pkg.GraphedGreedyDecoder(model, 2, 64).generate(ids, 10)
    assert a.shape == (2, 40)


def test_refusals(pkg, cuda):
    model = _model(cuda)
    with pytest.raises(ValueError, match="fuse_attention=True"):
        pkg.GraphedGreedyDecoder(model, 1, 64, kv_cache="int8")
    for kw in (dict(draft_tokens=4), dict(page_size=16)):
        with pytest.raises(ValueError, match="need kv_cache"):
            pkg.GraphedGreedyDecoder(model, 1, 64, **kw)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    for kw in (dict(draft_tokens=1), dict(draft_tokens=129), dict(kv_cache="int4"), dict(page_size=24)):
        with pytest.raises(ValueError):
            pkg.GraphedGreedyDecoder(model, 1, 64, **{"kv_cache": "int8", **kw})
    dec = pkg.GraphedGreedyDecoder(model, 2, 64, kv_cache="int8")
    with pytest.raises(ValueError, match="batch size"):
        dec.generate(_prompt(cuda, 1, 4), 4)
    with pytest.raises(ValueError, match="max_cache_len"):
        dec.generate(_prompt(cuda, 2, 60), 5)
    windowed = _model(cuda, use_sliding_window=True, sliding_window=16, max_window_layers=0)
    assert pkg.patch_model_with_fused_kernels(windowed, fuse_attention=True)["attention"] == 0


def test_a_ragged_prompt_over_a_used_cache(pkg, cuda):
    """More tokens than tree_attention takes, padding behind the shorter row, over slots that hold NaN from before."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    cache = pkg.DecoderCache.allocate(model, 2, 256, "16bit")
    for c in cache.layers:
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    ids, at = _prompt(cuda, 2, 200), torch.arange(200, device=cuda).expand(2, 200)
    cache.positions, cache.prompt = at, True
    cache.new_lens = torch.tensor([200, 150], dtype=torch.int32, device=cuda)
    with torch.inference_mode():
        logits = model(ids, past_key_values=cache.as_past(), position_ids=at, use_cache=True).logits.float()
        whole = model(ids).logits.float()
        short = model(ids[1:, :150]).logits.float()
        cache.tree_mask = torch.zeros((2, 200, 200), dtype=torch.bool, device=cuda)
        with pytest.raises(ValueError, match="a tree has at most 128"):
            model(ids, past_key_values=cache.as_past(), position_ids=at, use_cache=True)
    assert (logits[0] - whole[0]).abs().max().item() <= LOGIT_TOL["16bit"]
    assert (logits[1, :150] - short[0]).abs().max().item() <= LOGIT_TOL["16bit"]


@pytest.mark.parametrize("draft", [None, 6])
def test_a_model_that_builds_masks(pkg, cuda, draft):
    """HF's eager attention gets a causal mask with every step, which HF cannot build while a stream is captured."""
    model = _model(cuda)
    model.set_attn_implementation("eager")
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = torch.cat((_prompt(cuda, 1, 40, period=7), _prompt(cuda, 1, 40, seed=13)))
    dec = pkg.GraphedGreedyDecoder(model, 2, 120, use_graph=False, kv_cache="16bit", draft_tokens=draft)
    out, logits = dec.generate(ids, 20, return_logits=True)
    _check(pkg, model, dec, ids, out, logits, "16bit", f"eager draft {draft}")
