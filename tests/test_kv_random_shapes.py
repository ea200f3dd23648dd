"""Random shapes: a prompt appended, a draft appended behind it and attended to, the accepted branch moved together,
the next token attended to -- over pages in any order, some of them missing, against the 64-bit form."""
import random

import pytest
import torch

import kv_oracle as K

pytestmark = pytest.mark.gpu


def _rows(rng, g, batch, tokens, heads, d, dtype):
    """[batch, tokens, heads, d] on the GPU, contiguous or a view of something larger."""
    kind = rng.choice(("plain", "fused", "transposed", "odd"))
    if kind == "fused":  # a projection's output, other heads beside
        return torch.randn((batch, tokens, heads + 3, d), generator=g).to(dtype).cuda()[:, :, 1:heads + 1]
    if kind == "transposed":
        return torch.randn((batch, heads, tokens, d), generator=g).to(dtype).cuda().transpose(1, 2)
    if kind == "odd":  # rows that do not begin on 16 bytes
        return torch.randn((batch, tokens, heads, d + 3), generator=g).to(dtype).cuda()[..., 1:d + 1]
    return torch.randn((batch, tokens, heads, d), generator=g).to(dtype).cuda()


@pytest.mark.parametrize("seed", range(24))
def test_a_run(pkg, cuda, seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    kind, dtype = rng.choice(("16bit", "int8", "e4m3")), rng.choice((torch.float16, torch.bfloat16))
    batch, kvh, group, d = rng.randint(1, 5), rng.randint(1, 4), rng.randint(1, 9), 16 * rng.randint(1, 16)
    page = 16 * rng.choice((1, 1, 2, 3, 4, 5, 16))
    lens = [rng.choice((0, 1, 15, 16, 17, 31, 64, rng.randint(0, 300))) for _ in range(batch)]
    tokens = rng.choice((1, 2, 5, rng.randint(1, 40)))
    print(f"seed {seed}: {kind} {dtype} batch {batch} heads {kvh} x {group} d {d} page {page} lens {lens} tokens {tokens}",
          flush=True)
    per = (max(lens) + tokens + page) // page
    table, pages = K.shuffled_table(batch, per, 1, seed)
    if rng.random() < 0.3:  # pages that are not there
        table[rng.randrange(batch), rng.randrange(per)] = rng.choice((-1, pages, 2 ** 31 - 1))
    cache = K.make_cache(pkg, kind, dtype, (pages, kvh, page, d), table, seed + 1)
    half = rng.randint(1, d // 2)
    turn = dict(inv_freq=(1e4 ** (-torch.arange(half) / half)).float().cuda(), interleaved=rng.random() < 0.4, scale=1.1)
    pos = torch.arange(max(lens) + tokens + 1).cuda()

    # the prompt: slots 0 .. lens - 1, the rest of a row padding
    n = max(1, max(lens))
    pkg.kv_cache_append(cache, _rows(rng, g, batch, n, kvh, d, dtype), _rows(rng, g, batch, n, kvh, d, dtype),
                        K.ints([0] * batch), new_lens=K.ints(lens), positions=pos[:n], **turn)
    # the draft
    new = [rng.randint(0, tokens) for _ in range(batch)]
    at = torch.tensor(lens).cuda()[:, None] + pos[:tokens]
    q = pkg.kv_cache_append(cache, _rows(rng, g, batch, tokens, kvh, d, dtype), _rows(rng, g, batch, tokens, kvh, d, dtype),
                            K.ints(lens), new_lens=K.ints(new), q=_rows(rng, g, batch, tokens, kvh * group, d, dtype),
                            positions=at, **turn)
    mask = K.random_tree(batch, tokens, seed) if rng.random() < 0.7 else None
    out = pkg.tree_attention(q, cache, K.ints(lens), new_lens=K.ints(new), tree_mask=None if mask is None else mask.cuda())
    K.close(out, *K.attention(q, cache, lens, new=new, mask=mask))
    # some of it stays
    kept = [sorted(rng.sample(range(m), rng.randint(0, m))) for m in new]
    count = [len(k) for k in kept]
    most = max(1, max(count))
    held = [[K.place(cache, b, lens[b] + i) for i in k] for b, k in enumerate(kept)]
    before = [None if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    pkg.kv_cache_keep(cache, K.ints(lens), torch.tensor([k + [0] * (most - len(k)) for k in kept], dtype=torch.int32).cuda(),
                      K.ints(count))
    for b in range(batch):
        for i, was in enumerate(held[b]):
            now = K.place(cache, b, lens[b] + i)
            if was is None or now is None:
                continue
            for old, t in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
                if t is not None:
                    assert torch.equal(t[now[0], :, now[1]].float(), old[was[0], :, was[1]].float())
    # and the next token follows
    lens = [a + b for a, b in zip(lens, count)]
    q = pkg.kv_cache_append(cache, _rows(rng, g, batch, 1, kvh, d, dtype), _rows(rng, g, batch, 1, kvh, d, dtype),
                            K.ints(lens), q=_rows(rng, g, batch, 1, kvh * group, d, dtype),
                            positions=torch.tensor(lens).cuda()[:, None], **turn)
    K.close(pkg.tree_attention(q, cache, K.ints(lens)), *K.attention(q, cache, lens))
