"""Writing, reading and compacting the paged cache on the GPU against plain forms, exactly where the formula is exact."""
import pytest
import torch

import kv_oracle as K

pytestmark = pytest.mark.gpu

FORMATS = ["16bit", "int8", "e4m3"]


def _new(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _freq(pairs):
    return (1e6 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))).float()


def _snapshot(cache):
    return [None if t is None else (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).clone()
            for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def _same(a, b):
    """Bit for bit, NaN included."""
    def bits(t):
        return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])
    return a is b is None or torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,tokens,hq,kvh,d,page,lens,new,rotary,interleaved", [
    (1, 1, 12, 2, 128, 16, [0], None, 128, False),
    (3, 5, 14, 2, 64, 16, [0, 14, 33], None, 64, False),
    (2, 9, 6, 3, 96, 48, [47, 5], [9, 4], 24, True),
    (2, 20, 0, 5, 80, 32, [31, 0], [0, 20], 40, False),
    (1, 3, 8, 1, 256, 16, [60], None, 256, True),
    (1, 4, 2, 2, 16, 16, [3], None, 10, False),
    (2, 600, 3, 1, 64, 64, [1, 100], None, 0, False)])
def test_append_then_read(pkg, cuda, kind, dtype, batch, tokens, hq, kvh, d, page, lens, new, rotary, interleaved):
    per = (max(lens) + tokens + page - 1) // page
    table, pages = K.shuffled_table(batch, per, 2, 5)
    cache = K.make_cache(pkg, kind, dtype, (pages, kvh, page, d), table, 7)
    before = _snapshot(cache)
    k, v, q = (_new((batch, tokens, h, d), dtype, 11 + i) for i, h in enumerate((kvh, kvh, hq)))
    f = _freq(rotary // 2)
    pos = torch.tensor(lens)[:, None] + torch.arange(tokens)
    turn = dict(positions=pos.to(cuda), inv_freq=f.to(cuda), interleaved=interleaved, scale=1.25) if rotary else {}
    got_q = pkg.kv_cache_append(cache, k.to(cuda), v.to(cuda), K.ints(lens), new_lens=None if new is None else K.ints(new),
                                q=q.to(cuda) if hq and rotary else None, **turn)
    if hq and rotary:
        K.close(got_q, *K.rotary(q, pos, f, 1.25, interleaved))
    else:
        assert got_q is None
    kr, kb = K.rotary(k, pos, f, 1.25, interleaved) if rotary else (k.double(), torch.zeros(k.shape).double())
    after = _snapshot(cache)
    touched = torch.zeros((pages, page), dtype=torch.bool)
    for b in range(batch):
        for t in range(tokens if new is None else new[b]):
            p, at = K.place(cache, b, lens[b] + t)
            touched[p, at] = True
            if kind == "16bit":
                assert torch.equal(cache.v[p, :, at].cpu(), v[b, t])
                K.close(cache.k[p, :, at], kr[b, t], kb[b, t])
                continue
            code, scale = K.encode(v[b, t].float(), pkg.KV_FORMATS[kind])  # the same formula: the same bits
            assert torch.equal(cache.v[p, :, at].cpu().float(), code.float())
            assert torch.equal(cache.v_scale[p, :, at].cpu(), scale)
            # rotated keys: within half a step of their value, the largest of a row setting the step
            step = cache.k_scale[p, :, at].cpu().double()
            top = kr[b, t].abs().amax(-1)
            assert ((step - (top / K.TOP[pkg.KV_FORMATS[kind]]).clamp(min=1e-8)).abs() <= step * 1e-6).all()
            value = cache.k[p, :, at].cpu().float().double() * step[:, None]
            half = 0.5 * step[:, None] if kind == "int8" else (kr[b, t].abs() * 2.0 ** -4).clamp(min=2.0 ** -10 * step[:, None])
            # the quotient, at most 127, is rounded (2^-24) before it is rounded to a code: near a tie the code may be
            # the one beyond, at most 127 * 2^-24 of a step further off = 1.52e-5 halves (e4m3: |y| 2^-24 = 2^-20 halves)
            assert ((value - kr[b, t]).abs() - half * (1 + 1.6e-5) - kb[b, t]).max().item() <= 0
    for was, now in zip(before, after):  # nothing else was written
        if was is not None:
            kept = ~touched[:, None].expand(pages, kvh, page).to(cuda)
            assert torch.equal(was[kept], now[kept])
    # reading back: code * scale rounded once, zeros from the end on
    end = [n + (tokens if new is None else new[b]) for b, n in enumerate(lens)]
    start = [max(0, n - 2) for n in lens]
    rk, rv = pkg.kv_cache_read(cache, K.ints(end), tokens + 3, start=K.ints(start), dtype=dtype)
    assert rk.shape == rv.shape == (batch, kvh, tokens + 3, d)
    for b in range(batch):
        for i in range(tokens + 3):
            at = K.place(cache, b, start[b] + i) if start[b] + i < end[b] else None
            for got, pool, scale in ((rk, cache.k, cache.k_scale), (rv, cache.v, cache.v_scale)):
                want = torch.zeros((kvh, d), dtype=dtype, device=cuda)
                if at is not None:
                    x = pool[at[0], :, at[1]].float()
                    want = (x if scale is None else x * scale[at[0], :, at[1], None]).to(dtype)
                assert torch.equal(got[b, :, i], want)


@pytest.mark.parametrize("kind", FORMATS)
def test_slots_without_a_place(pkg, cuda, kind):
    """Page numbers of -1 and beyond the pool, slots beyond the table, negative lengths: nothing written, zeros read."""
    table = torch.tensor([[0, -1, 2], [1, 9, 1 << 30]])
    cache = K.make_cache(pkg, kind, torch.float16, (4, 2, 16, 64), table, 3)
    cases = [([16, 16], 16), ([32, 40], 8), ([48, 60], 5), ([2**31 - 3, 2**31 - 1], 9), ([-40, -7], 7)]
    for lens, tokens in cases:
        before = _snapshot(cache)
        x = _new((2, tokens, 2, 64), torch.float16, 4).to(cuda)
        pkg.kv_cache_append(cache, x, x, K.ints(lens))
        after = _snapshot(cache)
        for b in range(2):
            for t in range(tokens):
                at = K.place(cache, b, lens[b] + t)
                if at is not None:
                    for was, now in zip(before, after):
                        if was is not None:
                            was[at[0], :, at[1]] = now[at[0], :, at[1]]
        assert all(_same(a, b) for a, b in zip(before, after))
        rk, rv = pkg.kv_cache_read(cache, K.ints([2**31 - 1, 2**31 - 1]), tokens, start=K.ints(lens))
        for b in range(2):
            for t in range(tokens):
                if K.place(cache, b, lens[b] + t) is None:
                    assert not rk[b, :, t].any() and not rv[b, :, t].any()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_row_with_a_non_finite_value_reads_as_nan(pkg, cuda, kind, bad):
    cache = pkg.KVCache.allocate(1, 16, 2, 64, kind, device=cuda)
    x = _new((1, 3, 2, 64), torch.float16, 9)
    x[0, 1, 1, 37] = bad
    pkg.kv_cache_append(cache, x.to(cuda), x.to(cuda), K.ints([0]))
    for r in pkg.kv_cache_read(cache, K.ints([3]), 3):
        nan = r.isnan().cpu()
        assert nan[0, 1, 1].all() and nan.sum() == 64


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_zero_and_tiny_rows(pkg, cuda, kind):
    cache = pkg.KVCache.allocate(1, 16, 1, 64, kind, device=cuda)
    x = torch.zeros((1, 4, 1, 64), dtype=torch.float16)
    x[0, 1], x[0, 2, 0, 5], x[0, 3] = 6e-8, 65504.0, -65504.0
    pkg.kv_cache_append(cache, x.to(cuda), x.to(cuda), K.ints([0]))
    code, scale = K.encode(x.float(), pkg.KV_FORMATS[kind])
    assert torch.equal(cache.k[0, 0, :4].cpu().float(), code[0, :, 0].float())
    assert torch.equal(cache.k_scale[0, 0, :4].cpu(), scale[0, :, 0])


def test_strided_inputs(pkg, cuda):
    """k, v and q as slices of one projection, k with a stride that no packet fits (copied first)."""
    qkv = _new((2, 5, 16, 64), torch.bfloat16, 21).to(cuda)
    odd = _new((2, 5, 2 * 64 + 1), torch.bfloat16, 22).to(cuda)[..., 1:].unflatten(-1, (2, 64))
    f, pos = _freq(32).to(cuda), torch.arange(5, device=cuda)
    for k in (qkv[:, :, 12:14], odd, qkv[:, :, 12:14].transpose(1, 2).contiguous().transpose(1, 2)):
        a, b = (pkg.KVCache.allocate(2, 32, 2, 64, "int8", device=cuda) for _ in range(2))
        qa = pkg.kv_cache_append(a, k, qkv[:, :, 14:], K.ints([0, 3]), q=qkv[:, :, :12], positions=pos, inv_freq=f)
        qb = pkg.kv_cache_append(b, k.contiguous(), qkv[:, :, 14:].contiguous(), K.ints([0, 3]),
                                 q=qkv[:, :, :12].contiguous(), positions=pos, inv_freq=f)
        assert torch.equal(qa, qb) and all(_same(x, y) for x, y in zip(_snapshot(a), _snapshot(b)))


@pytest.mark.parametrize("kind", FORMATS)
@pytest.mark.parametrize("kvh,d,page", [(2, 128, 16), (3, 80, 48), (1, 256, 32), (1, 16, 16)])
def test_keep_any_order(pkg, cuda, kind, kvh, d, page):
    """Ascending paths, a reversal, repeats, all to themselves, negative entries, counts of 0 and beyond the row."""
    kept = [[0, 2, 5, 9], [3, 2, 1, 0], [1, 1, 1, 1], [0, 1, 2, 3], [-1, 4, -7, 2], [7, 6, 5, 4]]
    counts = [4, 4, 3, 4, 4, 0]
    lens = [0, 13, 30, 5, 47, 2]
    per = (max(lens) + 12 + page - 1) // page
    table, pages = K.shuffled_table(6, per, 1, 8)
    cache = K.make_cache(pkg, kind, torch.float16, (pages, kvh, page, d), table, 12)
    for n in (counts, None, [99] * 6):
        before = _snapshot(cache)
        pkg.kv_cache_keep(cache, K.ints(lens), K.ints(kept), None if n is None else K.ints(n))
        want = [None if t is None else t.clone() for t in before]
        for b in range(6):
            for i in range(4 if n is None else min(4, n[b])):
                if kept[b][i] < 0:
                    continue
                (p, at), (tp, tat) = K.place(cache, b, lens[b] + kept[b][i]), K.place(cache, b, lens[b] + i)
                for w, t in zip(want, before):
                    if t is not None:
                        w[tp, :, tat] = t[p, :, at]
        assert all(_same(a, b) for a, b in zip(_snapshot(cache), want))


def test_keep_128_and_slots_without_a_place(pkg, cuda):
    cache = K.make_cache(pkg, "int8", torch.float16, (20, 2, 16, 128), [list(range(10)) + [-1, 11, 12, 13, 14, 15]], 13)
    before = _snapshot(cache)
    kept = torch.randperm(140, generator=torch.Generator().manual_seed(1))[:128]
    pkg.kv_cache_keep(cache, K.ints([20]), K.ints([kept.tolist()]))
    want = [t.clone() for t in before]
    for i, j in enumerate(kept.tolist()):
        src, dst = K.place(cache, 0, 20 + j), K.place(cache, 0, 20 + i)
        if src and dst:
            for w, t in zip(want, before):
                w[dst[0], :, dst[1]] = t[src[0], :, src[1]]
    assert all(_same(a, b) for a, b in zip(_snapshot(cache), want))


def test_offsets_beyond_32_bits(pkg, cuda):
    """A pool of more than 4 GiB per side: the last pages are written, moved and read."""
    pages, page = 300_000, 16
    cache = pkg.KVCache(*(torch.zeros((pages, 8, page, 128), dtype=torch.uint8, device=cuda).view(torch.int8)
                          for _ in range(2)), K.ints([[pages - 1, pages - 2]]),
                        *(torch.zeros((pages, 8, page), device=cuda) for _ in range(2)))
    assert cache.k.numel() > 1 << 32
    x = _new((1, 20, 8, 128), torch.float16, 30).to(cuda)
    pkg.kv_cache_append(cache, x, x, K.ints([0]))
    pkg.kv_cache_keep(cache, K.ints([0]), K.ints([[19]]))
    rk, rv = pkg.kv_cache_read(cache, K.ints([20]), 20)
    code, scale = K.encode(x.float(), torch.int8)
    want = (code.float() * scale[..., None]).half().transpose(1, 2)
    want = torch.cat((want[:, :, 19:], want[:, :, 1:]), 2)
    assert torch.equal(rk, want) and torch.equal(rv, want)
    del cache
    torch.cuda.empty_cache()


def test_graph_replays_and_other_stream(pkg, cuda):
    """Append, keep and read captured once, replayed with other inputs and lengths, between eager calls."""
    caches = [pkg.KVCache.allocate(2, 64, 2, 64, "e4m3", device=cuda, page_size=16) for _ in range(2)]
    k, v, q = (torch.zeros((2, 4, h, 64), dtype=torch.float16, device=cuda) for h in (2, 2, 6))
    lens, pos = K.ints([0, 0]), torch.zeros((2, 4), dtype=torch.long, device=cuda)
    kept, n, f = K.ints([[0, 2], [1, 3]]), K.ints([2, 1]), _freq(32).to(cuda)

    def step(cache):
        out = pkg.kv_cache_append(cache, k, v, lens, q=q, positions=pos, inv_freq=f)
        pkg.kv_cache_keep(cache, lens, kept, n)
        return (out, *pkg.kv_cache_read(cache, lens + n, 8))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])
        step(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for i in range(4):
        for j, t in enumerate((k, v, q)):
            t.copy_(_new(t.shape, torch.float16, 50 + 3 * i + j))
        lens.copy_(K.ints([5 * i, 11 * i]))
        pos.copy_(lens[:, None].long() + torch.arange(4, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(_same(a, b) for a, b in zip(_snapshot(caches[0]), _snapshot(caches[1])))


def test_empty_calls(pkg, cuda):
    cache = pkg.KVCache.allocate(2, 32, 2, 64, "int8", device=cuda)
    x = torch.empty((2, 0, 2, 64), dtype=torch.float16, device=cuda)
    assert pkg.kv_cache_append(cache, x, x, K.ints([0, 0])) is None
    assert pkg.kv_cache_read(cache, K.ints([0, 0]), 0)[0].shape == (2, 2, 0, 64)
    pkg.kv_cache_keep(cache, K.ints([0, 0]), torch.empty((2, 0), dtype=torch.int32, device=cuda))


def test_refusals(pkg, cuda):
    cache = pkg.KVCache.allocate(2, 32, 2, 64, "int8", device=cuda)
    x = torch.zeros((2, 3, 2, 64), dtype=torch.float16, device=cuda)
    lens, pos, f = K.ints([0, 0]), torch.zeros((2, 3), dtype=torch.long, device=cuda), _freq(32).to(cuda)
    make = pkg.KVCache
    for args, kw, message in [
            ((cache, x.cpu(), x, lens), {}, "GPU"), ((cache, x.float(), x.float(), lens), {}, "fp16 or bf16"),
            ((cache, x, x.bfloat16(), lens), {}, "share a dtype"), ((cache, x, x[:, :2], lens), {}, "differ"),
            ((cache, x[:, :, :1], x[:, :, :1], lens), {}, "heads"), ((cache, x[:1], x[:1], lens[:1]), {}, "sequences"),
            ((cache, x, x, lens.long()), {}, "int32"), ((cache, x, x, lens.cpu()), {}, "seq_lens"),
            ((cache, x, x, lens), {"new_lens": lens[:1]}, "new_lens"), ((cache, x, x, lens), {"q": x}, "rotated"),
            ((cache, x, x, lens), {"inv_freq": f}, "together"),
            ((cache, x, x, lens), {"q": x[:, :2], "positions": pos, "inv_freq": f}, "does not fit"),
            ((make(cache.k, cache.v, cache.page_table), x, x, lens), {}, "needs k_scale"),
            ((make(cache.k, cache.v, cache.page_table.long(), cache.k_scale, cache.v_scale), x, x, lens), {}, "page_table"),
            ((make(cache.k.transpose(1, 2), cache.v.transpose(1, 2), cache.page_table, cache.k_scale, cache.v_scale), x, x,
              lens), {}, "contiguous"),
            ((make(cache.k, cache.v, cache.page_table, cache.k_scale[:1], cache.v_scale), x, x, lens), {}, "scales"),
            ((make(x, x, cache.page_table, cache.k_scale, cache.v_scale), x, x, lens), {}, "no scales"),
            ((make(x.float(), x.float(), cache.page_table), x, x, lens), {}, "cache dtype")]:
        with pytest.raises(AssertionError, match=message):
            pkg.kv_cache_append(*args, **kw)
    with pytest.raises(Exception, match="page_size must be a multiple of 16"):
        wide = torch.zeros((2, 3, 3, 64), dtype=torch.float16, device=cuda)
        pkg.kv_cache_append(make(x, x, cache.page_table), wide, wide, lens)  # pools of 3 heads and pages of 2
    sixteen = pkg.KVCache.allocate(2, 32, 2, 64, "16bit", torch.bfloat16, device=cuda)
    with pytest.raises(AssertionError, match="the cache torch.bfloat16"):
        pkg.kv_cache_append(sixteen, x, x, lens)
    with pytest.raises(AssertionError, match="the cache torch.bfloat16"):
        pkg.kv_cache_read(sixteen, lens, 2, dtype=torch.float16)
    with pytest.raises(AssertionError, match="tokens"):
        pkg.kv_cache_read(cache, lens, -1)
    with pytest.raises(AssertionError, match="kept"):
        pkg.kv_cache_keep(cache, lens, lens)
    with pytest.raises(Exception, match="max_kept <= 128"):
        pkg.kv_cache_keep(cache, lens, torch.zeros((2, 129), dtype=torch.int32, device=cuda))
