"""tree_attention on the GPU against its 64-bit form: lengths from nothing to long, masks that leave rows empty, and
values in places that nobody sees."""
import pytest
import torch

import kv_oracle as K

pytestmark = pytest.mark.gpu

FORMATS = ["16bit", "int8", "e4m3"]


def _q(shape, dtype, seed, std=2.0):
    return (std * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _case(pkg, kind, dtype, batch, tokens, hq, kvh, d, page, lens, seed=1):
    per = max(1, (max(lens) + tokens + page - 1) // page)
    table, pages = K.shuffled_table(batch, per, 2, seed)
    cache = K.make_cache(pkg, kind, dtype, (pages, kvh, page, d), table, seed + 1)
    return cache, _q((batch, tokens, hq, d), dtype, seed + 2).cuda()


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,tokens,hq,kvh,d,page,lens,tree", [
    (1, 1, 1, 1, 64, 16, [0], False),
    (1, 1, 12, 2, 128, 16, [777], False),
    (4, 1, 14, 2, 64, 16, [0, 1, 31, 300], False),
    (3, 5, 28, 4, 128, 48, [0, 47, 130], True),
    (2, 17, 6, 3, 96, 32, [64, 9], True),
    (2, 33, 10, 5, 80, 64, [63, 200], False),
    (1, 64, 8, 1, 256, 16, [40], True),
    (2, 128, 4, 4, 16, 256, [250, 0], True),
    (5, 3, 40, 8, 128, 16, [16, 32, 48, 15, 17], False),
    (1, 50, 28, 4, 128, 64, [100], True),
    (2, 3, 8, 1, 256, 32, [70, 5], True),
    (1, 20, 6, 1, 64, 32, [33], True),
    (1, 2, 32, 32, 32, 16, [1030], False)])
def test_matches_64_bit_form(pkg, cuda, kind, dtype, batch, tokens, hq, kvh, d, page, lens, tree):
    cache, q = _case(pkg, kind, dtype, batch, tokens, hq, kvh, d, page, lens)
    mask = K.random_tree(batch, tokens, 3) if tree else None
    out = pkg.tree_attention(q, cache, K.ints(lens), tree_mask=None if mask is None else mask.to(cuda))
    assert out.shape == q.shape and out.dtype == dtype
    K.close(out, *K.attention(q, cache, lens, mask=mask))
    again = pkg.tree_attention(q, cache, K.ints(lens), tree_mask=None if mask is None else mask.to(cuda))
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("lens,batch_pad", [([20011], 0), ([9000, 3, 511, 0], 0)])
def test_long_and_unequal_contexts(pkg, cuda, kind, lens, batch_pad):
    """Contexts that are split over workgroups, beside ones that are not."""
    cache, q = _case(pkg, kind, torch.bfloat16, len(lens), 2, 8, 2, 128, 64, lens)
    K.close(pkg.tree_attention(q, cache, K.ints(lens)), *K.attention(q, cache, lens))


@pytest.mark.parametrize("tokens,kind,d", [(20, "int8", 64), (12, "16bit", 128), (9, "e4m3", 256)])
def test_long_contexts_of_many_rows(pkg, cuda, tokens, kind, d):
    lens = [5000, 700]
    cache, q = _case(pkg, kind, torch.float16, 2, tokens, 12, 2, d, 48, lens)
    mask = K.random_tree(2, tokens, 9)
    K.close(pkg.tree_attention(q, cache, K.ints(lens), tree_mask=mask.to(cuda)), *K.attention(q, cache, lens, mask=mask))


@pytest.mark.parametrize("tokens", [1, 40])
def test_more_than_64_sequences(pkg, cuda, tokens):
    """Contexts of 0 to 400 slots of 150 sequences: the plan goes over the lengths in several rounds."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    lens[:3], lens[63:66], lens[149] = [0, 0, 400], [1, 399, 0], 400
    new = torch.randint(0, tokens + 1, (150,), generator=g).tolist()
    cache, q = _case(pkg, "int8", torch.float16, 150, tokens, 2, 1, 32, 16, lens)
    pick = [0, 1, 2, 63, 64, 65, 100, 128, 149]
    out = pkg.tree_attention(q, cache, K.ints(lens), new_lens=K.ints(new))
    part = pkg.KVCache(cache.k, cache.v, cache.page_table[pick], cache.k_scale, cache.v_scale)
    K.close(out[pick], *K.attention(q[pick], part, [lens[i] for i in pick], [new[i] for i in pick]))
    # all of them against the same sequences in batches of their own
    for i in range(0, 150, 50):
        part = pkg.KVCache(cache.k, cache.v, cache.page_table[i:i + 50], cache.k_scale, cache.v_scale)
        one = pkg.tree_attention(q[i:i + 50], part, K.ints(lens[i:i + 50]), new_lens=K.ints(new[i:i + 50]))
        # other splits of the same sums: fp32 rounding and one step of fp16
        assert (one.float() - out[i:i + 50].float()).abs().max().item() <= 2.0 ** -9


def test_without_a_workspace(pkg, cuda):
    """The C call without scratch memory: every sequence and head in one workgroup, the same result up to the order of
    the sums."""
    import ctypes
    import importlib
    L = importlib.import_module("llm-inference-optimizer_amd._lib")
    for tokens, lens in ((1, [3000, 17, 0]), (30, [900, 65, 0])):
        cache, q = _case(pkg, "int8", torch.float16, 3, tokens, 6, 2, 128, 32, lens)
        c = L.KvCacheStruct(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                            cache.page_table.data_ptr(), cache.page_table.shape[1], cache.page_table.shape[1],
                            *cache.k.shape, L.KV_INT8)
        n = K.ints(lens)
        lib = L.load()
        assert lib.mi355_tree_attention_workspace(ctypes.byref(c), 3, tokens, 6) > 0
        out = torch.full_like(q, float("nan"))
        strides = (ctypes.c_int64 * 3)(*q.stride()[:3])
        assert lib.mi355_tree_attention_fwd(ctypes.byref(c), q.data_ptr(), out.data_ptr(), n.data_ptr(), None, None, 0, 0,
                                            3, tokens, 6, strides, 128 ** -0.5, L.F16, None, 0,
                                            L.stream_handle(q.device)) == 0
        K.close(out, *K.attention(q, cache, lens))


@pytest.mark.parametrize("kind", FORMATS)
def test_rows_that_see_nothing_and_padding(pkg, cuda, kind):
    """Empty mask rows without a context get zeros; with one, the context alone; padding gets zeros."""
    lens, new = [0, 0, 37, 5], [6, 3, 6, 0]
    cache, q = _case(pkg, kind, torch.float16, 4, 6, 4, 2, 64, 16, lens)
    mask = K.random_tree(4, 6, 4)
    mask[0, 2] = False
    mask[2, 3] = False
    mask[1] = False
    out = pkg.tree_attention(q, cache, K.ints(lens), new_lens=K.ints(new), tree_mask=mask.to(cuda))
    K.close(out, *K.attention(q, cache, lens, new, mask))
    assert not out[0, 2].any() and not out[1].any() and not out[3].any() and out[2, 3].any()


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_unseen_values_have_no_influence(pkg, cuda, kind, d):
    """NaN, infinities and largest values in slots behind the last token, in padding tokens, and in drafted tokens of
    other branches -- keys, values and scales -- leave a row's bits as they are."""
    batch, tokens, lens, new = 2, 6, [37, 3], [6, 4]
    cache, q = _case(pkg, kind, torch.float16, batch, tokens, 6, 2, d, 16, lens)
    mask = torch.eye(tokens, dtype=torch.bool).expand(batch, tokens, tokens).clone()
    mask[:, 1:, 0] = True   # token 0 is everyone's parent but token 5's; nobody else sees tokens 1 .. 5
    mask[:, 5] = False
    mask[:, 5, 5] = True
    args = dict(new_lens=K.ints(new), tree_mask=mask.to(cuda))
    want = pkg.tree_attention(q, cache, K.ints(lens), **args)
    K.close(want, *K.attention(q, cache, lens, new, mask))
    for bad in (float("nan"), float("inf"), float("-inf"), 65504.0):
        hit = pkg.KVCache(*(None if t is None else t.clone() for t in cache.tensors()))
        for b in range(batch):
            for s in [lens[b] + 1, lens[b] + 3] + list(range(lens[b] + new[b], lens[b] + 16)):
                at = K.place(cache, b, s)
                if at is None:
                    continue
                for pool, scale in ((hit.k, hit.k_scale), (hit.v, hit.v_scale)):
                    if kind == "16bit":
                        pool[at[0], :, at[1], ::3] = bad
                    else:
                        scale[at[0], :, at[1]] = bad
                        if kind == "e4m3":
                            pool.view(torch.uint8)[at[0], :, at[1], ::3] = 0x7f  # e4m3's NaN
        got = pkg.tree_attention(q, hit, K.ints(lens), **args)
        ok = torch.ones((batch, tokens), dtype=torch.bool, device=cuda)
        ok[:, [1, 3]] = False  # they see themselves
        assert torch.equal(got[ok], want[ok]), bad
        assert not got[ok].isnan().any()
        if bad != bad:
            assert got[0, 1].isnan().any(-1).all() and got[0, 3].isnan().any(-1).all()


def test_seen_values_that_are_not_finite(pkg, cuda):
    """A visible NaN key makes its rows NaN, a visible NaN value its column; rows whose scores are all -infinity get
    zeros."""
    cache, q = _case(pkg, "16bit", torch.float16, 1, 2, 2, 1, 64, 16, [5])
    p, at = K.place(cache, 0, 6)
    for pool, rows in ((cache.k, slice(None)), (cache.v, 7)):
        was = pool[p, 0, at, 7].item()
        pool[p, 0, at, 7] = float("nan")
        out = pkg.tree_attention(q, cache, K.ints([5]))
        assert out[0, 1][:, rows].isnan().all() and not out[0, 0].isnan().any()
        if rows == 7:
            assert out[0, 1].isnan().sum() == 2
        pool[p, 0, at, 7] = was
    q[:] = 1.0
    cache.k[:] = float("-inf")
    assert not pkg.tree_attention(q, cache, K.ints([5])).any()


@pytest.mark.parametrize("kind", FORMATS)
def test_pages_that_are_not_there(pkg, cuda, kind):
    """Pages of -1 or beyond the pool are not attended to, nor are slots beyond the table."""
    table = torch.tensor([[0, -1, 2, 5], [99, 1, 3, -1], [-1, -1, -1, -1]])
    cache = K.make_cache(pkg, kind, torch.bfloat16, (6, 2, 16, 64), table, 3)
    q = _q((3, 4, 4, 64), torch.bfloat16, 5).to(cuda)
    for lens in ([60, 60, 60], [62, 10, 0], [64, 1000, 2**31 - 1], [-5, 0, -2**31]):
        K.close(pkg.tree_attention(q, cache, K.ints(lens)), *K.attention(q, cache, lens))


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("tokens", [3, 40])
def test_scale_of_zero_and_below(pkg, cuda, kind, tokens):
    """With a scale of 0 every slot that is seen weighs the same, and one that is not still nothing."""
    lens = [70, 0, 33]
    cache, q = _case(pkg, kind, torch.bfloat16, 3, tokens, 4, 2, 64, 16, lens)
    for scale in (0.0, -0.0, -0.3):
        K.close(pkg.tree_attention(q, cache, K.ints(lens), scale=scale), *K.attention(q, cache, lens, scale=scale))


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("tokens,length", [(1, 40), (1, 700), (20, 700), (70, 700)])
def test_scores_near_the_lowest_number(pkg, cuda, kind, tokens, length):
    """Scores of -10^33 and below are scores like others: the least negative one takes all the weight, and equal ones
    share it -- a product that is rounded for the maximum has to be the same one in the exponent."""
    cache, q = _case(pkg, kind, torch.bfloat16, 1, tokens, 2, 1, 64, 16, [length])
    quantised = cache.k_scale is not None
    unit = 1.0 if quantised else 1e17
    q.zero_()
    q[..., 0] = 1.7e17
    rows = torch.zeros(cache.k.shape, dtype=torch.float32, device=cuda)
    rows[..., 0] = -3 * unit
    page, place = cache.page_table[0, 1].item(), 3  # slot 19, before the new tokens
    rows[page, 0, place, 0] = -unit
    cache.k.copy_(rows.to(cache.k.dtype))
    if quantised:
        cache.k_scale.fill_(1.1e17)
        v = cache.v[page, 0, place].float() * cache.v_scale[page, 0, place]
    else:
        v = cache.v[page, 0, place].float()
    out = pkg.tree_attention(q, cache, K.ints([length]), scale=0.3)
    # weight 1, whose product with the scale is off by 2^-16 (two bf16 parts), and one rounding to bf16
    assert ((out.float() - v).abs() <= v.abs() * (2.0 ** -8 + 2.0 ** -15)).all()
    # the same score everywhere: the values' mean
    cache.k.copy_((rows * 0 + (rows != 0) * (-unit)).to(cache.k.dtype))
    first = torch.zeros((1, tokens, tokens), dtype=torch.bool, device=cuda)
    out = pkg.tree_attention(q, cache, K.ints([length]), tree_mask=first, scale=0.3)
    k, values = pkg.kv_cache_read(cache, K.ints([length]), length, dtype=torch.bfloat16)
    mean, spread = values.double().mean(2)[:, :, None], values.double().abs().mean(2)[:, :, None]
    # read rounds every value (2^-8), the weights are off by 2^-16, the sum by 700 * 2^-24, the result by 2^-8
    assert ((out.double().transpose(1, 2) - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -7.9 * spread).all()


def test_large_scores_and_scale(pkg, cuda):
    """Scores of some hundreds: the exponentials' range, a running maximum that keeps rising, a scale of its own."""
    lens = [600, 100]
    cache, q = _case(pkg, "int8", torch.float16, 2, 3, 6, 2, 64, 32, lens)
    q *= 8
    ramp = torch.linspace(0.01, 3, cache.k_scale.shape[2], device=cuda)
    cache.k_scale *= ramp
    for scale in (1.0, 0.01, -0.5):
        K.close(pkg.tree_attention(q, cache, K.ints(lens), scale=scale), *K.attention(q, cache, lens, scale=scale))


def test_strided_queries_and_masks(pkg, cuda):
    lens = [20, 50]
    cache, _ = _case(pkg, "int8", torch.float16, 2, 5, 6, 2, 64, 16, lens)
    qkv = _q((2, 5, 10, 64), torch.float16, 9).to(cuda)
    odd = _q((2, 5, 6 * 64 + 1), torch.float16, 10).to(cuda)[..., 1:].unflatten(-1, (6, 64))
    one = K.random_tree(1, 5, 6)
    masks = [one.to(cuda), one[0].to(cuda), one[0].T.contiguous().T.to(cuda), one.to(cuda).expand(2, 5, 5),
             torch.nn.functional.pad(one, (0, 3)).to(cuda)[..., :5]]
    for q in (qkv[:, :, 2:8], odd, qkv[:, :, :6].transpose(1, 2).contiguous().transpose(1, 2)):
        want = pkg.tree_attention(q.contiguous(), cache, K.ints(lens), tree_mask=one.expand(2, 5, 5).contiguous().to(cuda))
        for mask in masks:
            assert torch.equal(pkg.tree_attention(q, cache, K.ints(lens), tree_mask=mask), want)


def test_offsets_beyond_32_bits(pkg, cuda):
    pages, page = 300_000, 16
    cache = pkg.KVCache(*(torch.zeros((pages, 8, page, 128), dtype=torch.uint8, device=cuda).view(torch.int8)
                          for _ in range(2)), K.ints([[pages - 1, pages - 2, pages - 3]]),
                        *(torch.zeros((pages, 8, page), device=cuda) for _ in range(2)))
    x = _q((1, 40, 8, 128), torch.float16, 30, 1.0).to(cuda)
    small = pkg.KVCache.allocate(1, 48, 8, 128, "int8", device=cuda, page_size=16)
    for c in (cache, small):
        pkg.kv_cache_append(c, x, x, K.ints([0]))
    q = _q((1, 2, 16, 128), torch.float16, 31).to(cuda)
    assert torch.equal(pkg.tree_attention(q, cache, K.ints([38])), pkg.tree_attention(q, small, K.ints([38])))
    del cache
    torch.cuda.empty_cache()


def test_graphs_share_a_pool_and_other_streams(pkg, cuda):
    """Two captured steps of different sizes in one memory pool, replayed in turn with other lengths and contents, and
    eager calls on a side stream at the same time."""
    cases = [_case(pkg, "int8", torch.float16, 2, 1, 12, 2, 128, 16, [4000, 4000]),
             _case(pkg, "e4m3", torch.bfloat16, 1, 7, 14, 2, 64, 32, [3000], seed=5)]
    lens = [K.ints([4000, 4000]), K.ints([3000])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for (c, q), n in zip(cases, lens):
            pkg.tree_attention(q, c, n)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for (c, q), n in zip(cases, lens):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(pkg.tree_attention(q, c, n))
        pool = graph.pool()
        graphs.append(graph)
    for i in range(4):
        lens[0].copy_(K.ints([1 + 1333 * i, 4000 - 900 * i]))
        lens[1].copy_(K.ints([3000 - 999 * i]))
        for (c, q), n in zip(cases, lens):
            q.copy_(_q(q.shape, q.dtype, 70 + i))
        for which in ((0, 1), (1, 0))[i % 2]:
            graphs[which].replay()
            torch.cuda.synchronize()
            (c, q), n = cases[which], lens[which]
            want = pkg.tree_attention(q, c, n)
            assert torch.equal(outs[which], want)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = pkg.tree_attention(q, c, n)
            here = pkg.tree_attention(q, c, n)
            torch.cuda.synchronize()
            assert torch.equal(other, want) and torch.equal(here, want)


def test_empty_calls(pkg, cuda):
    cache = pkg.KVCache.allocate(2, 32, 2, 64, "int8", device=cuda)
    q = torch.empty((2, 0, 4, 64), dtype=torch.float16, device=cuda)
    assert pkg.tree_attention(q, cache, K.ints([0, 0])).shape == q.shape


def test_refusals(pkg, cuda):
    cache = pkg.KVCache.allocate(2, 32, 2, 64, "int8", device=cuda)
    q, lens = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=cuda), K.ints([0, 0])
    mask = torch.zeros((3, 3), dtype=torch.bool, device=cuda)
    for args, kw, message in [
            ((q.cpu(), cache, lens), {}, "GPU"), ((q.float(), cache, lens), {}, "fp16 or bf16"),
            ((q[0], cache, lens), {}, r"\[batch"), ((q[..., :32], cache, lens), {}, "heads"),
            ((q[:, :, :3], cache, lens), {}, "heads"), ((q[:1], cache, lens[:1]), {}, "sequences"),
            ((q, cache, lens.long()), {}, "int32"), ((q, cache, lens), {"new_lens": lens[:1]}, "new_lens"),
            ((q, cache, lens), {"tree_mask": mask.int()}, "tree_mask"), ((q, cache, lens), {"tree_mask": mask[:2]}, "tree_mask"),
            ((q, cache, lens), {"tree_mask": mask.expand(3, 3, 3)}, "tree_mask"),
            ((q, cache, lens), {"tree_mask": mask.cpu()}, "tree_mask")]:
        with pytest.raises(AssertionError, match=message):
            pkg.tree_attention(*args, **kw)
    with pytest.raises(Exception, match="tokens <= 128"):
        pkg.tree_attention(torch.zeros((2, 129, 4, 64), dtype=torch.float16, device=cuda), cache, lens)


def _without_workspace(q, cache, lens):
    """The C call without scratch memory, over a 16-bit cache."""
    import ctypes
    import importlib
    L = importlib.import_module("llm-inference-optimizer_amd._lib")
    batch, tokens, heads, d = q.shape
    width = cache.page_table.shape[1]
    c = L.KvCacheStruct(cache.k.data_ptr(), cache.v.data_ptr(), None, None, cache.page_table.data_ptr(), width, width,
                        *cache.k.shape, L.KV_16BIT)
    n, out = K.ints(lens), torch.full_like(q, float("nan"))
    strides = (ctypes.c_int64 * 3)(*q.stride()[:3])
    assert L.load().mi355_tree_attention_fwd(ctypes.byref(c), q.data_ptr(), out.data_ptr(), n.data_ptr(), None, None, 0,
                                             0, batch, tokens, heads, strides, 1.0,
                                             L.F16 if q.dtype == torch.float16 else L.BF16, None, 0,
                                             L.stream_handle(q.device)) == 0
    torch.cuda.synchronize()
    return out


def _sink_scores(pattern, n, nats):
    """Scores of n slots, and which of them have a value."""
    at = torch.arange(n)
    if pattern in ("first", "last"):  # one slot stands out and says nothing
        sink = at == (0 if pattern == "first" else n - 1)
        return torch.where(sink, 0.0, -float(nats)), ~sink
    if pattern in ("falling", "rising"):  # by 5 nats every 192 slots, the strongest 768 of them without a value
        step = at // 192 if pattern == "falling" else (n - 1 - at) // 192
        return -5.0 * step, step >= 4
    # every other 64 slots stand out
    return torch.where(at // 64 % 2 == 0, 0.0, -float(nats)), at // 64 % 2 == 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pattern,nats", [("first", 12), ("first", 15), ("first", 18), ("last", 18), ("falling", 5),
                                          ("rising", 5), ("every other", 18)])
@pytest.mark.parametrize("tokens,heads,d", [(1, 3, 64), (5, 4, 128), (3, 9, 256), (10, 4, 64), (30, 4, 128), (9, 6, 256)])
def test_small_weights_that_matter(pkg, cuda, dtype, pattern, nats, tokens, heads, d):
    """The slots with the largest weights have values of 0, so that weights 12 to 18 nats below the largest (and, falling
    or rising, below those before or behind them) make the result: the bound counts their 16 bits like any others'."""
    n = 4000
    cache, q = _case(pkg, "16bit", dtype, 1, tokens, heads, 1, d, 32, [n])
    score, valued = _sink_scores(pattern, n, nats)
    q.zero_()
    q[..., 0] = 1.0
    q[:, :, 1::2, 0] = 0.75  # other rows, other distances
    slot = torch.arange(n)
    page, place = cache.page_table[0, (slot // 32).to(cuda)].long(), (slot % 32).to(cuda)
    cache.k.zero_()
    cache.k[page, 0, place, 0] = score.to(dtype).to(cuda)
    last = torch.arange(n, n + tokens)  # the new tokens: as far below as the pattern's least
    cache.k[cache.page_table[0, (last // 32).to(cuda)].long(), 0, (last % 32).to(cuda), 0] = float(score.min())
    cache.v.abs_().clamp_(0.25, 1.0)
    cache.v[page, 0, place] *= valued[:, None].to(dtype).to(cuda)
    want = K.attention(q, cache, [n], scale=1.0)
    K.close(pkg.tree_attention(q, cache, K.ints([n]), scale=1.0), *want)
    K.close(_without_workspace(q, cache, [n]), *want)


def _expect_values(out, q, cache, lens, mask=None):
    """Elements with a visible NaN or both infinities are NaN, those with one infinity are it, others as ever; codes
    whose scale is not finite count as NaN."""
    held = [t.clone() if t is not None else None for t in cache.tensors()]
    k, v, _, ks, vs = held
    codes = v.float()
    bad = ~codes.isfinite() | (~vs.isfinite()[..., None] if vs is not None else False)
    value = torch.where(codes.isfinite(), float("nan"), codes) if vs is not None else codes
    (v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v)[bad] = 0
    if vs is not None:
        vs[~vs.isfinite()] = 0
    clean = type(cache)(*held)
    want, bound = K.attention(q, clean, lens, mask=mask)
    got = K.cpu(out)
    batch, tokens, hq, _ = q.shape
    special = torch.zeros(want.shape, dtype=torch.float32)
    for b in range(batch):
        for s in range(lens[b] + tokens):
            at = K.place(cache, b, s)
            row = torch.where(bad[at[0], :, at[1]], value[at[0], :, at[1]], 0.0).cpu()  # [kv_heads, d]
            if not row.any():
                continue
            row = row.repeat_interleave(hq // row.shape[0], 0)
            for t in range(tokens):
                j = s - lens[b]
                if j < 0 or (mask[b, t, j] if mask is not None else j <= t):
                    special[b, t] += row
    plain = special == 0
    K.close(torch.where(plain, got, 0), torch.where(plain, want, 0.0), torch.where(plain, bound, 0.0))
    assert torch.equal(got.float()[~plain].nan_to_num(12345.0, 1.0, -1.0), special[~plain].nan_to_num(12345.0, 1.0, -1.0))


@pytest.mark.parametrize("kind,dtype", [("16bit", torch.float16), ("16bit", torch.bfloat16), ("int8", torch.float16),
                                        ("e4m3", torch.bfloat16)])
@pytest.mark.parametrize("tokens,heads,d", [(1, 4, 64), (1, 6, 128), (10, 6, 128), (20, 6, 64), (30, 8, 128), (12, 10, 256)])
@pytest.mark.parametrize("length", [90, 2000])
def test_visible_infinities(pkg, cuda, kind, dtype, tokens, heads, d, length):
    """An infinite value that a row sees makes that element infinite -- in slots that all rows see as in drafted ones,
    in one piece or many, at a large weight or a small one."""
    lens = [length, length // 2]
    cache, q = _case(pkg, kind, dtype, 2, tokens, heads, 2, d, 16, lens)
    inf, nan = float("inf"), float("nan")
    for b, s, e, x in [(0, 0, 0, inf), (0, length // 2, 1, -inf), (0, length - 1, 2, inf), (0, 3, 3, inf),
                       (0, length - 20, 3, -inf), (0, 40, 4, nan), (0, length, 5, inf), (1, 7, d - 1, inf),
                       (1, 7, d - 2, -inf), (1, length // 4, d - 1, inf)]:
        page, at = K.place(cache, b, s)
        if kind == "16bit":
            cache.v[page, 1, at, e] = x
        elif s % 2:  # the whole row
            cache.v_scale[page, 1, at] = x
        elif kind == "e4m3":
            cache.v.view(torch.uint8)[page, 1, at, e] = 0x7f
    mask = K.random_tree(2, tokens, 3)
    out = pkg.tree_attention(q, cache, K.ints(lens), tree_mask=mask.to(cuda))
    _expect_values(out, q, cache, lens, mask)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("nats", [60, 200])
def test_a_visible_infinity_of_a_weight_that_vanishes(pkg, cuda, tokens, nats):
    """The weight of the infinite value is beyond 32 bits of exponent (not beyond 64), in another piece than the rest."""
    n = 3000
    cache, q = _case(pkg, "16bit", torch.bfloat16, 1, tokens, 2, 1, 64, 32, [n])
    q.zero_()
    q[..., 0] = 8.0
    cache.k.zero_()
    for s in (5, 2900):
        page, at = K.place(cache, 0, s)
        cache.k[page, 0, at, 0] = -float(nats)  # 8 nats / sqrt(64)
        cache.v[page, 0, at, s % 7] = float("inf")
    _expect_values(pkg.tree_attention(q, cache, K.ints([n])), q, cache, [n])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [144, 208, 240])
@pytest.mark.parametrize("tokens,length", [(1, 40), (5, 600), (24, 600)])
def test_non_finite_first_elements_of_heads_that_fill_no_tile(pkg, cuda, dtype, d, tokens, length):
    """Lanes beyond the last element hold zeros, whatever the unit's first elements are."""
    cache, q = _case(pkg, "16bit", dtype, 1, tokens, 4, 2, d, 16, [length])
    for s, x in ((length // 3, float("inf")), (length, float("nan")), (length - 1, -float("inf"))):
        page, at = K.place(cache, 0, s)
        cache.v[page, 0, at, s % 8] = x
    mask = K.random_tree(1, tokens, 3)
    _expect_values(pkg.tree_attention(q, cache, K.ints([length]), tree_mask=mask.to(cuda)), q, cache, [length], mask)
