"""shared_prefix_attention against the 64-bit form, and against tree_attention over tables that say the same."""
import math

import pytest
import torch
from kv_oracle import close, ints, make_cache, random_tree, shuffled_table
from shared_oracle import attention, members

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _setup(pkg, kind, dtype, heads, sizes, prefix, own, tokens, page, seed, junk=False):
    """A cache whose groups share whole pages of their prefix; the entry of a page that the prefix ends in is the first
    member's for the prefix and each member's own behind it.  junk: members' entries for the prefix name nothing."""
    hq, kvh, d = heads
    batch = sum(sizes)
    longest = max(p for p in prefix) + max(own) + tokens
    per = -(-longest // page)
    table, pages = shuffled_table(batch, per, 3, seed)
    table = table.clone()
    first = 0
    for size, p in zip(sizes, prefix):
        table[first:first + size, :p // page] = table[first, :p // page].clone()
        if junk:
            table[first + 1:first + size, :p // page] = -1
        first += size
    cache = make_cache(pkg, kind, dtype, (pages, kvh, page, d), table, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((batch, tokens, hq, d), generator=g) * 1.5).to(dtype).cuda()
    lens = [p + own[sum(sizes[:i]) + j] for i, p in enumerate(prefix) for j in range(sizes[i])]
    starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    return cache, q, lens, starts


HEADS = [(14, 2, 64), (12, 2, 128), (4, 4, 32), (6, 1, 96), (8, 2, 256), (5, 1, 80), (40, 8, 128)]


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", HEADS)
def test_heads_and_formats(pkg, cuda, kind, dtype, heads):
    sizes, prefix = [3, 1, 2], [75, 40, 16]
    own = [0, 9, 33, 5, 1, 70]
    cache, q, lens, starts = _setup(pkg, kind, dtype, heads, sizes, prefix, own, 1, 16, 3)
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), ints(starts))
    close(out, *attention(q, cache, lens, prefix, starts))


@pytest.mark.parametrize("tokens", [2, 5, 17, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("kind,dtype", [("16bit", F16), ("16bit", BF16), ("int8", BF16), ("e4m3", F16)])
def test_several_tokens(pkg, cuda, tokens, tree, kind, dtype):
    sizes, prefix, own = [4, 2], [130, 37], [0, 3, 50, 20, 9, 64]
    cache, q, lens, starts = _setup(pkg, kind, dtype, (6, 2, 64), sizes, prefix, own, tokens, 32, 5)
    mask = random_tree(6, tokens, 7) if tree else None
    new = [tokens, max(0, tokens - 1), 0, tokens, 1, tokens]
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), ints(starts), new_lens=ints(new),
                                      tree_mask=mask.cuda() if tree else None)
    value, bound = attention(q, cache, lens, prefix, starts, new, mask)
    close(out, value, bound)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 63, 64, 65, 127, 129, 500])
def test_prefix_ends(pkg, cuda, page, prefix):
    """Prefixes that end anywhere in a page and a tile; entries that the members have for them are not looked at."""
    sizes, own = [5], [0, 1, 15, 40, 100]
    for kind in ("16bit", "int8"):
        cache, q, lens, starts = _setup(pkg, kind, F16, (4, 2, 64), sizes, [prefix], own, 1, page, prefix, junk=True)
        out = pkg.shared_prefix_attention(q, cache, ints(lens), ints([prefix]))
        close(out, *attention(q, cache, lens, [prefix]))


@pytest.mark.parametrize("size,tokens,heads", [(1, 1, (8, 2, 64)), (3, 1, (28, 4, 128)), (33, 1, (4, 4, 64)), (64, 1, (14, 2, 64)),
                                               (20, 3, (16, 2, 128)), (9, 1, (16, 1, 256)), (130, 1, (2, 1, 64)), (5, 40, (6, 2, 96))])
@pytest.mark.parametrize("kind", ["16bit", "int8"])
def test_many_rows(pkg, cuda, size, tokens, heads, kind):
    """Row blocks that a group fills once, several times and partly, over prefixes that are split."""
    own = [(7 * i) % 90 for i in range(2 * size)]
    prefix = [1500, 700]
    cache, q, lens, _ = _setup(pkg, kind, BF16, heads, [size, size], prefix, own, tokens, 64, 11)
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix))
    close(out, *attention(q, cache, lens, prefix))


def test_lengths_that_do_not_fit(pkg, cuda):
    """Sequences with less than the prefix in the cache (a padded batch's rows of length 0 among them), prefixes beyond
    everything or negative, sequences of no group, empty groups, boundaries outside the batch."""
    sizes, prefix, own = [6, 2], [100, 64], [0, 5, 20, 1, 40, 9, 30, 2]
    cache, q, lens, starts = _setup(pkg, "int8", F16, (4, 2, 64), sizes, prefix, own, 2, 16, 13)
    for lens2 in (lens, [0, 3, 50, 99, 100, 101, 64, 10], [0] * 8, [-5, 10 ** 9, 100, 3, 2 ** 31 - 1, 0, 17, 16]):
        for prefix2 in (prefix, [10 ** 9, 16], [-3, 0], [2 ** 31 - 1, 2 ** 31 - 1]):
            out = pkg.shared_prefix_attention(q, cache, ints(lens2), ints(prefix2), ints(starts))
            close(out, *attention(q, cache, lens2, prefix2, starts))
    for groups, prefix2 in (([2, 5, 7], [100, 30]), ([0, 0, 8], [30, 100]), ([3, 3, 3], [50, 60]), ([-4, 4, 100], [90, 33]),
                            ([6, 2, 8], [40, 50]), ([1, 4], [70]), ([0], [])):
        out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix2), ints(groups))
        close(out, *attention(q, cache, lens, prefix2, groups))


def test_nothing_shared_is_tree_attention(pkg, cuda):
    cache, q, lens, _ = _setup(pkg, "int8", BF16, (12, 2, 128), [4], [300], [0, 50, 100, 7], 3, 32, 17)
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints([]))
    value, bound = attention(q, cache, lens, [])
    close(out, value, bound)
    close(pkg.tree_attention(q, cache, ints(lens)), value, bound)
    assert pkg.shared_prefix_attention(q[:0], pkg.KVCache(cache.k, cache.v, cache.page_table[:0], cache.k_scale, cache.v_scale),
                                       ints([]), ints([])).shape == (0, 3, 12, 128)
    assert pkg.shared_prefix_attention(q[:, :0], cache, ints(lens), ints([300])).shape == (4, 0, 12, 128)


@pytest.mark.parametrize("kind,dtype", [("16bit", F16), ("16bit", BF16), ("int8", F16), ("e4m3", BF16)])
def test_pages_that_are_not_there(pkg, cuda, kind, dtype):
    """Holes in the first member's prefix and in own pages: their slots are not attended to."""
    sizes, prefix, own = [3, 2], [200, 90], [40, 60, 5, 33, 80]
    cache, q, lens, starts = _setup(pkg, kind, dtype, (4, 2, 64), sizes, prefix, own, 2, 16, 19)
    cache.page_table[0, 3] = -1
    cache.page_table[0, 7:9] = 10 ** 6
    cache.page_table[1, 13] = -1
    cache.page_table[3] = -1
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), ints(starts))
    close(out, *attention(q, cache, lens, prefix, starts))
    cache.page_table.fill_(-1)
    assert (pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), ints(starts)) == 0).all()


@pytest.mark.parametrize("kind,dtype", [("16bit", F16), ("16bit", BF16), ("int8", F16), ("e4m3", BF16)])
@pytest.mark.parametrize("size", [2, 24])
def test_what_nobody_sees_may_be_anything(pkg, cuda, kind, dtype, size):
    """NaN and infinities behind the lengths, in masked drafts, in the members' own entries of the prefix and in pages
    of nobody."""
    prefix, own, tokens = [150], [(5 * i) % 37 for i in range(size)], 3
    cache, q, lens, _ = _setup(pkg, kind, dtype, (6, 2, 64), [size], prefix, own, tokens, 16, 23)
    mask = random_tree(size, tokens, 3)
    want = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), tree_mask=mask.cuda())
    close(want, *attention(q, cache, lens, prefix, None, None, mask))
    seen = torch.zeros(cache.k.shape[0], 16, dtype=torch.bool)
    table = cache.page_table.cpu()
    for s in range(150):
        seen[table[0, s // 16], s % 16] = True
    for b in range(size):
        for s in range(150, lens[b] + tokens):
            seen[table[b, s // 16], s % 16] = True
    at = (~seen).cuda()[:, None, :].expand(cache.k.shape[:3])
    if kind == "16bit":
        for pool, bad in ((cache.k, math.nan), (cache.v, math.inf)):
            pool.masked_fill_(at[..., None], bad)
    else:
        for scale, bad in ((cache.k_scale, math.inf), (cache.v_scale, math.nan)):
            scale.masked_fill_(at, bad)
    got = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), tree_mask=mask.cuda())
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [3, 40])
@pytest.mark.parametrize("slot", [0, 77, 149])
def test_infinite_values_of_the_prefix(pkg, cuda, dtype, size, slot):
    """An infinity in the prefix reaches its element of every member that sees it, and no other element."""
    prefix, own = [150], [(5 * i) % 37 for i in range(size)]
    cache, q, lens, _ = _setup(pkg, "16bit", dtype, (6, 2, 64), [size], prefix, own, 1, 16, 29)
    lens[1] = 60  # does not see slots from 60 on
    want = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix)).clone()
    page = int(cache.page_table[0, slot // 16])
    cache.v[page, 1, slot % 16, 5] = math.inf
    cache.v[page, 0, slot % 16, 63] = math.nan
    got = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix))
    for b in range(size):
        if slot < min(lens[b], 150):
            assert (got[b, 0, 3:, 5] == math.inf).all() and got[b, 0, :3, 63].isnan().all()
            got[b, 0, 3:, 5], got[b, 0, :3, 63] = want[b, 0, 3:, 5], want[b, 0, :3, 63]
    assert torch.equal(got, want)


def test_a_scale_that_is_not_finite(pkg, cuda):
    prefix, own = [100], [5, 9, 0, 20]
    cache, q, lens, _ = _setup(pkg, "int8", F16, (4, 2, 64), [4], prefix, own, 1, 16, 31)
    cache.v_scale[int(cache.page_table[0, 2]), 1, 3] = math.inf
    got = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix))
    assert got[:, :, 2:].isnan().all() and not got[:, :, :2].isnan().any()


def test_large_scores_and_far_apart_maxima(pkg, cuda):
    """The prefix outweighs the own slots, or they it, by more than 32 bits hold: the sums are joined by their maxima."""
    for factor in (0.02, 50.0):
        cache, q, lens, _ = _setup(pkg, "16bit", BF16, (4, 2, 64), [5], [300], [40, 3, 0, 9, 100], 1, 32, 37)
        for b in range(5):
            for s in range(300, lens[b] + 1):
                cache.k[int(cache.page_table[b, s // 32]), :, s % 32] *= factor
        out = pkg.shared_prefix_attention(q * 4, cache, ints(lens), ints([300]))
        close(out, *attention(q * 4, cache, lens, [300]))


def test_strided_queries_and_scale(pkg, cuda):
    cache, q, lens, starts = _setup(pkg, "int8", F16, (4, 2, 64), [3, 2], [90, 50], [3, 20, 9, 0, 60], 2, 16, 41)
    wide = torch.zeros((5, 4, 2, 128), dtype=F16, device="cuda")
    wide[..., 8:72] = q.transpose(1, 2)
    out = pkg.shared_prefix_attention(wide[..., 8:72].transpose(1, 2), cache, ints(lens), ints([90, 50]), ints(starts), scale=0.3)
    close(out, *attention(q, cache, lens, [90, 50], starts, scale=0.3))
    odd = torch.zeros((5, 2, 4, 67), dtype=F16, device="cuda")
    odd[..., 3:] = q
    assert torch.equal(pkg.shared_prefix_attention(odd[..., 3:], cache, ints(lens), ints([90, 50]), ints(starts), scale=0.3), out)


def test_long_prefix(pkg, cuda):
    """20000 slots for 48 sequences: many pieces of every row."""
    own = [(37 * i) % 300 for i in range(48)]
    for kind, dtype in (("16bit", BF16), ("int8", F16)):
        cache, q, lens, _ = _setup(pkg, kind, dtype, (7, 1, 128), [48], [20000], own, 1, 64, 43)
        out = pkg.shared_prefix_attention(q, cache, ints(lens), ints([20000]))
        close(out, *attention(q, cache, lens, [20000]))


@pytest.mark.parametrize("kind", ["16bit", "int8"])
def test_graphs_and_streams(pkg, cuda, kind):
    """Two captured graphs and eager calls, lengths that change between replays; equal calls give equal bits."""
    sizes, prefix, own = [10, 6], [400, 150], [(11 * i) % 80 for i in range(16)]
    cache, q, lens, starts = _setup(pkg, kind, F16, (14, 2, 64), sizes, prefix, own, 2, 32, 47)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        static = [q.clone(), ints(lens), ints(prefix), ints(starts)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pkg.shared_prefix_attention(static[0], cache, *static[1:])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pkg.shared_prefix_attention(static[0], cache, *static[1:])
        graphs.append((graph, static, out))
    for i in range(5):
        args = [q * (1 + 0.1 * i), ints([max(0, n - 20 * i) for n in lens]), ints([max(0, p - 7 * i) for p in prefix]), ints(starts)]
        want = pkg.shared_prefix_attention(args[0], cache, *args[1:])
        for graph, static, _ in graphs:
            for to, new in zip(static, args):
                to.copy_(new)
            graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = pkg.shared_prefix_attention(args[0], cache, *args[1:])
        torch.cuda.synchronize()
        assert torch.equal(again, want) and all(torch.equal(out, want) for _, _, out in graphs)


def test_members_helper():
    assert members(6, 2, None) == [(0, 3), (3, 3)] and members(6, 2, [1, 4, 9]) == [(1, 3), (4, 2)]
