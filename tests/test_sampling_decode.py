"""GraphedSamplingDecoder: kv_cache_reserve, kv_cache_append, shared_prefix_attention and sample_tokens together, as a
decode step uses them, against an independent prefill of the decoded sequences into HF's DynamicCache."""
import math

import pytest
import torch

from decode_check import reference_pass, sharpen_attention
from shared_oracle import sample

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")

LAYERS, VOCAB = 4, 512
# as tests/test_cached_decode.py has them: what the cache's formats do to 4 layers' logits of about 4
LOGIT_TOL = {"16bit": 0.05, "int8": 0.2, "e4m3": 1.0}


def _model(cuda, seed=3, dtype=torch.float16, heads=4, kv_heads=2, hidden=256, vocab=VOCAB):
    cfg = transformers.Qwen2Config(vocab_size=vocab, hidden_size=hidden, intermediate_size=512,
                                   num_hidden_layers=LAYERS, num_attention_heads=heads, num_key_value_heads=kv_heads,
                                   max_position_embeddings=4096, rms_norm_eps=1e-6, tie_word_embeddings=True,
                                   attn_implementation="sdpa", initializer_range=0.06,
                                   rope_parameters={"rope_theta": 1e6, "rope_type": "default"})
    torch.manual_seed(seed)
    with torch.device(cuda):
        m = transformers.Qwen2ForCausalLM(cfg)
    m = m.to(dtype).eval()
    sharpen_attention(m, 1.5)
    return m


def _prompt(cuda, batch, length, vocab=VOCAB, seed=11):
    return torch.randint(0, vocab, (batch, length), generator=torch.Generator().manual_seed(seed)).to(cuda)


def _reference(model, ids, out):
    """Logits that predict each new token, [batch, samples, new, vocab]."""
    n, m, length = out.shape
    flat = out.view(n * m, length)
    p = ids.shape[1]
    logits, _ = reference_pass(model, flat[:, :p], flat[:, p:])
    return logits.view(n, m, length - p, -1)


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("length", [5, 32, 77, 200])  # less than a page, whole pages, a part, a prompt beyond the tree's
def test_draws_from_the_model(pkg, cuda, kind, length):
    """The probabilities that tokens were drawn with are the model's, as an independent pass over each whole
    continuation has them: a page, position or prefix gone wrong is off by order one."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True, fuse_residual=True)
    ids = _prompt(cuda, 2, length)
    dec = pkg.GraphedSamplingDecoder(model, 2, 5, 260, kv_cache=kind, page_size=32, temperature=0.8)
    u = torch.rand((2, 5, 40), generator=torch.Generator().manual_seed(length))
    out, logs = dec.generate(ids, 40, uniform=u, return_logprobs=True)
    assert out.shape == (2, 5, length + 40) and logs.shape == (2, 5, 40) and dec._graph is not None
    assert torch.equal(out[:, :, :length], ids[:, None].expand(2, 5, length))
    assert len({tuple(row) for row in out[0].tolist()}) == 5  # other numbers, other texts
    want = torch.log_softmax(_reference(model, ids, out) / 0.8, -1).gather(-1, out[:, :, length:, None])[..., 0]
    worst = (logs - want).abs().max().item()
    print(f"{kind} {length}: logarithms off by {worst:.3g}")
    assert worst <= 2 * LOGIT_TOL[kind] / 0.8
    # the same numbers again, through the captured graph and eagerly: the same tokens
    assert torch.equal(dec.generate(ids, 40, uniform=u), out)
    eager = pkg.GraphedSamplingDecoder(model, 2, 5, 260, kv_cache=kind, page_size=32, temperature=0.8, use_graph=False)
    again, logs2 = eager.generate(ids, 40, uniform=u, return_logprobs=True)
    assert torch.equal(again, out) and torch.equal(logs2, logs)


def test_tokens_are_those_of_the_definition(pkg, cuda):
    """Every draw, from the reference's logits by the definition, but where rounding of the logits may decide."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = _prompt(cuda, 2, 50)
    settings = dict(temperature=0.9, top_k=20, top_p=0.9, min_p=0.02)
    dec = pkg.GraphedSamplingDecoder(model, 2, 4, 120, page_size=16, **settings)
    u = torch.rand((2, 4, 30), generator=torch.Generator().manual_seed(5))
    out = dec.generate(ids, 30, uniform=u)
    ref = _reference(model, ids, out).cpu()
    same = 0
    for b in range(2):
        for s in range(4):
            for i in range(30):
                token, _, near = sample(ref[b, s, i], u[b, s, i].item(), **settings)
                got = int(out[b, s, 50 + i])
                same += got == token
                assert got == token or near < 0.05, (b, s, i)
    print(f"{same} of 240 draws the same")
    assert same >= 0.9 * 240


def test_greedy_samples_are_the_greedy_decoder_s(pkg, cuda):
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = _prompt(cuda, 3, 60)
    out = pkg.GraphedSamplingDecoder(model, 3, 3, 120, page_size=32, temperature=0.0).generate(ids, 40)
    ref = _reference(model, ids, out)
    picked = ref.gather(-1, out[:, :, 60:, None])[..., 0]
    assert (ref.amax(-1) - picked).max().item() <= 2 * LOGIT_TOL["16bit"]  # the largest but for near-ties
    assert torch.equal(out[:, 0], out[:, 1]) and torch.equal(out[:, 0], out[:, 2])


def test_settings_per_sample_and_a_large_vocabulary(pkg, cuda):
    model = _model(cuda, vocab=151936)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = _prompt(cuda, 1, 40, vocab=151936)
    dec = pkg.GraphedSamplingDecoder(model, 1, 4, 100, kv_cache="int8", temperature=torch.tensor([0.0, 0.7, 1.0, 1.5]),
                                     top_k=torch.tensor([0, 1, 50, 0]), top_p=0.95)
    for seed in (1, 2):
        u = torch.rand((1, 4, 30), generator=torch.Generator().manual_seed(seed))
        out, logs = dec.generate(ids, 30, uniform=u, return_logprobs=True)
        assert out.min() >= 0 and out.max() < 151936
        assert torch.equal(out[0, 0], out[0, 1]) and (logs[0, :2] == 0).all()  # greedy, and the first of one
        assert torch.equal(dec.generate(ids, 30, uniform=u), out)
    one = dec.generate(ids, 1, uniform=u[:, :, :1])
    assert torch.equal(one, out[:, :, :41])


def test_pages(pkg, cuda):
    """What a generation takes of the pool: prompts once, the rest per sample; a pool of just that is enough, one page
    less is refused; its pages are free again for the next."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    probe = pkg.GraphedSamplingDecoder(model, 2, 6, 300, page_size=16)
    assert probe.pages_needed(100, 30) == 2 * (6 + 6 * 3)  # 129 slots: 6 whole pages, 3 more
    tight = pkg.GraphedSamplingDecoder(model, 2, 6, 300, page_size=16, pages=probe.pages_needed(100, 30))
    ids = _prompt(cuda, 2, 100)
    u = torch.rand((2, 6, 30), generator=torch.Generator().manual_seed(3))
    want = probe.generate(ids, 30, uniform=u)
    for _ in range(2):
        assert torch.equal(tight.generate(ids, 30, uniform=u), want)
    table = tight.table.view(2, 6, -1)
    used = table[table >= 0]
    assert len(used.unique()) == tight.pages and (table[:, :, :6] == table[:, :1, :6]).all()
    with pytest.raises(ValueError, match="pages"):
        tight.generate(ids, 60)
    assert torch.equal(tight.generate(ids[:, :90], 20, uniform=u[:, :, :20]), probe.generate(ids[:, :90], 20, uniform=u[:, :, :20]))


def test_refusals(pkg, cuda):
    model = _model(cuda)
    with pytest.raises(ValueError, match="fuse_attention"):
        pkg.GraphedSamplingDecoder(model, 1, 2, 64)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    for kw in (dict(batch_size=0, samples=2), dict(batch_size=1, samples=0), dict(batch_size=1, samples=2, page_size=24),
               dict(batch_size=1, samples=2, pages=0), dict(batch_size=1, samples=2, kv_cache="int4")):
        with pytest.raises(ValueError):
            pkg.GraphedSamplingDecoder(model, max_cache_len=64, **kw)
    dec = pkg.GraphedSamplingDecoder(model, 2, 2, 64, page_size=16)
    ids = _prompt(cuda, 2, 10)
    for call in (lambda: dec.generate(ids[:1], 5), lambda: dec.generate(ids, 0), lambda: dec.generate(ids, 55),
                 lambda: dec.generate(ids, 5, uniform=torch.rand(2, 2, 4))):
        with pytest.raises(ValueError):
            call()
    assert math.isfinite(float(dec.generate(ids, 5, return_logprobs=True)[1].sum()))


@pytest.mark.parametrize("kind", ["16bit", "int8"])
def test_prompts_read_once_or_for_each_sample(pkg, cuda, kind):
    """Both attentions draw from the model, and a decoder follows the prompt's length from one to the other and back."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True, fuse_residual=True)
    u = torch.rand((2, 5, 40), generator=torch.Generator().manual_seed(71))
    outs = {}
    for share in (True, False):
        dec = pkg.GraphedSamplingDecoder(model, 2, 5, 260, kv_cache=kind, page_size=32, temperature=0.8, share_prefix=share)
        for length in (77, 200):
            ids = _prompt(cuda, 2, length)
            out, logs = dec.generate(ids, 40, uniform=u, return_logprobs=True)
            assert (dec.cache.shared_prefix is not None) == share
            want = torch.log_softmax(_reference(model, ids, out) / 0.8, -1).gather(-1, out[:, :, length:, None])[..., 0]
            assert (logs - want).abs().max().item() <= 2 * LOGIT_TOL[kind] / 0.8
            outs[share, length] = out
    dec = pkg.GraphedSamplingDecoder(model, 2, 5, 260, kv_cache=kind, page_size=32, temperature=0.8)
    dec._shares = lambda length: length > 100
    for length in (77, 200, 77):
        assert torch.equal(dec.generate(_prompt(cuda, 2, length), 40, uniform=u), outs[length > 100, length])
    assert len(dec._graphs) == 2


def test_which_attention(pkg, cuda):
    """The rule: what the prompts' continuations would read, keys and values of 2 heads of 64 with scales, 272 bytes a token."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    dec = pkg.GraphedSamplingDecoder(model, 4, 16, 4096, kv_cache="int8", pages=64)
    assert not dec._shares(64 * 2 ** 20 // (64 * 272) - 1) and dec._shares(64 * 2 ** 20 // (64 * 272) + 1)
    assert not pkg.GraphedSamplingDecoder(model, 64, 1, 4096, kv_cache="int8", pages=64)._shares(4096)
