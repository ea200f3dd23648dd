"""kv_cache_reserve and kv_slot_map against their definitions, entry by entry: whole numbers, which have to be equal."""
import pytest
import torch
from shared_oracle import reserve, slot_map

pytestmark = pytest.mark.gpu


def _ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _cache(pkg, cuda, table, pages, page_size):
    pool = torch.zeros((pages, 1, page_size, 16), dtype=torch.float16, device=cuda)
    return pkg.KVCache(pool, pool, table if torch.is_tensor(table) else _ints(table, cuda))


def _random(batch, width, pages, page_size, seed, shared=True):
    """A table with pages, holes, numbers outside the pool and pages that several rows name; lengths that end anywhere."""
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(max(pages, batch * width), generator=g)[:batch * width].view(batch, width)
    table = torch.where(table < pages, table, -1)
    holes = torch.rand((batch, width), generator=g)
    table = torch.where(holes < 0.2, -1, torch.where(holes > 0.97, pages + 3, table))
    if shared and batch > 1:
        table[1, :width // 2] = table[0, :width // 2]
    lens = torch.randint(-3, width * page_size + 1, (batch,), generator=g)
    new = torch.randint(-2, 2 * page_size, (batch,), generator=g)
    lens[torch.rand((batch,), generator=g) < 0.2] = 0
    return table.tolist(), lens.tolist(), new.tolist()


SIZES = [(1, 1, 1, 16), (1, 5, 3, 32), (2, 3, 40, 16), (7, 13, 64, 48), (33, 9, 500, 16), (5, 200, 900, 16),
         (64, 65, 4096, 16), (3, 64, 4097, 256), (130, 70, 12000, 64), (700, 3, 2000, 16), (2100, 40, 90000, 16)]


@pytest.mark.parametrize("batch,width,pages,page_size", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve(pkg, cuda, batch, width, pages, page_size, in_place):
    for seed in (1, 2):
        table, lens, new = _random(batch, width, pages, page_size, seed)
        cache = _cache(pkg, cuda, table, pages, page_size)
        want, missing = reserve(table, pages, page_size, lens, new)
        out = None if in_place else torch.full((batch, width), 77, dtype=torch.int32, device=cuda)
        got, short = pkg.kv_cache_reserve(cache, _ints(lens, cuda), _ints(new, cuda), out=out)
        assert got is (cache.page_table if in_place else out) or got.data_ptr() == (cache.page_table if in_place else out).data_ptr()
        assert got.tolist() == want and short.tolist() == missing
        if not in_place:
            assert cache.page_table.tolist() == table


def test_reserve_without_new_lengths(pkg, cuda):
    cache = _cache(pkg, cuda, [[-1, -1], [-1, -1]], 3, 16)
    assert pkg.kv_cache_reserve(cache, _ints([17, 16], cuda))[1].tolist() == [0, 0]
    assert cache.page_table.tolist() == [[0, 1], [2, -1]]


def test_pages_run_out(pkg, cuda):
    """The first sequences get what there is; lengths beyond the table and beyond 2^31 slots count as missing."""
    cache = _cache(pkg, cuda, [[-1] * 4 for _ in range(3)], 5, 16)
    table, missing = pkg.kv_cache_reserve(cache, _ints([48, 48, 16], cuda), _ints([0, 0, 0], cuda))
    assert table.tolist() == [[0, 1, 2, -1], [3, 4, -1, -1], [-1] * 4] and missing.tolist() == [0, 1, 1]
    big = 2 ** 31 - 1
    _, missing = pkg.kv_cache_reserve(cache, _ints([big, 0, 0], cuda), _ints([big, 0, 0], cuda))
    assert cache.page_table.tolist() == [[0, 1, 2, 3], [-1] * 4, [-1] * 4]
    assert missing.tolist() == [-(-2 * big // 16) - 4, 0, 0]


def test_shared_pages_live_as_long_as_a_row_needs_them(pkg, cuda):
    cache = _cache(pkg, cuda, [[0, 1, 2], [0, 1, 3]], 5, 16)
    pkg.kv_cache_reserve(cache, _ints([0, 40], cuda))  # sequence 0 ended: page 2 is free, 0 and 1 are not
    assert cache.page_table.tolist() == [[-1] * 3, [0, 1, 3]]
    pkg.kv_cache_reserve(cache, _ints([33, 40], cuda))
    assert cache.page_table.tolist() == [[2, 4, -1], [0, 1, 3]]


def test_reserve_strided_tables(pkg, cuda):
    """Every other row of a table, and a table whose rows lie in a larger buffer; neighbours stay as they were."""
    table, lens, new = _random(6, 10, 100, 16, 3)
    want, missing = reserve(table, 100, 16, lens, new)
    wide = torch.full((12, 15), 55, dtype=torch.int32, device=cuda)
    view = wide[::2, 2:12]
    view.copy_(torch.tensor(table))
    got, short = pkg.kv_cache_reserve(_cache(pkg, cuda, view, 100, 16), _ints(lens, cuda), _ints(new, cuda))
    assert got.tolist() == want and short.tolist() == missing
    assert (wide[1::2] == 55).all() and (wide[:, :2] == 55).all() and (wide[:, 12:] == 55).all()
    # a new table that overlaps the old one, shifted by a column
    both = torch.full((6, 11), 55, dtype=torch.int32, device=cuda)
    both[:, :10] = torch.tensor(table)
    pkg.kv_cache_reserve(_cache(pkg, cuda, both[:, :10], 100, 16), _ints(lens, cuda), _ints(new, cuda), out=both[:, 1:])
    assert both[:, 1:].tolist() == want
    # transposed tables are read, but not written in place
    turned = _ints(table, cuda).t().contiguous().t()
    cache = _cache(pkg, cuda, turned, 100, 16)
    got, _ = pkg.kv_cache_reserve(cache, _ints(lens, cuda), _ints(new, cuda), out=torch.empty_like(both[:, :10]).contiguous())
    assert got.tolist() == want
    with pytest.raises(AssertionError, match="contiguous rows"):
        pkg.kv_cache_reserve(cache, _ints(lens, cuda))


def test_reserve_empty_batch(pkg, cuda):
    cache = _cache(pkg, cuda, torch.empty((0, 4), dtype=torch.int32, device=cuda), 5, 16)
    table, missing = pkg.kv_cache_reserve(cache, _ints([], cuda))
    assert table.shape == (0, 4) and missing.shape == (0,)


@pytest.mark.parametrize("batch,width,pages,page_size", [(1, 1, 1, 16), (3, 5, 9, 32), (70, 12, 700, 48), (1500, 4, 5000, 16),
                                                         (9000, 3, 20000, 16)])
def test_slot_map(pkg, cuda, batch, width, pages, page_size):
    table, lens, new = _random(batch, width, pages, page_size, 5)
    lens = [min(n, width * page_size - 5) for n in lens]  # the last tokens of some lie beyond the table
    total = sum(max(0, m) for m in new)
    cache = _cache(pkg, cuda, table, pages, page_size)
    for tokens in sorted({total, total + 100, max(1, total // 2), 1, 0}):
        got = pkg.kv_slot_map(cache, _ints(lens, cuda), _ints(new, cuda), tokens)
        assert [t.dtype for t in got] == [torch.int64, torch.int32, torch.int64]
        want = slot_map(table, pages, page_size, lens, new, tokens)
        assert list(zip(*(t.tolist() for t in got))) == want


def test_slot_map_places_what_append_writes(pkg, cuda):
    """The slots are those that kv_cache_append writes to and kv_cache_read reads from."""
    lens, new, page = [5, 0, 30], [9, 20, 3], 16
    cache = pkg.KVCache.allocate(3, 48, 2, 32, "16bit", torch.float16, cuda, page)
    cache.page_table.fill_(-1)
    pkg.kv_cache_reserve(cache, _ints(lens, cuda), _ints(new, cuda))
    k = torch.randn(3, 20, 2, 32, device=cuda).half()
    pkg.kv_cache_append(cache, k, -k, _ints(lens, cuda), new_lens=_ints(new, cuda))
    slots, owners, positions = pkg.kv_slot_map(cache, _ints(lens, cuda), _ints(new, cuda), sum(new))
    t = positions - _ints(lens, cuda)[owners.long()]
    assert torch.equal(cache.k[slots // page, :, slots % page], k[owners.long(), t])
    assert torch.equal(cache.v[slots // page, :, slots % page], -k[owners.long(), t])


def test_positions_beyond_32_bits(pkg, cuda):
    big = 2 ** 31 - 1
    cache = _cache(pkg, cuda, [[0, 1]], 2, 16)
    slots, owners, positions = pkg.kv_slot_map(cache, _ints([big], cuda), _ints([big], cuda), 5)
    assert positions.tolist() == [big + i for i in range(5)] and slots.tolist() == [-1] * 5 and owners.tolist() == [0] * 5


def test_pages_in_a_graph_and_on_another_stream(pkg, cuda):
    """A captured step that grows its sequences: replays follow the lengths; two graphs with eager calls between."""
    page, width = 16, 40
    side = torch.cuda.Stream()

    def make():
        cache = _cache(pkg, cuda, [[-1] * width for _ in range(5)], 120, page)
        return cache, _ints([0, 3, 15, 16, 200], cuda), _ints([1, 2, 3, 4, 5], cuda)

    graphs = []
    for _ in range(2):
        cache, lens, new = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pkg.kv_cache_reserve(cache, lens, new)
        torch.cuda.current_stream().wait_stream(side)
        cache.page_table.fill_(-1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            missing = pkg.kv_cache_reserve(cache, lens, new)[1]
            slots = pkg.kv_slot_map(cache, lens, new, 15)
            lens.add_(new)
        cache.page_table.fill_(-1)
        graphs.append((graph, cache, lens, new, missing, slots))
    eager_cache, eager_lens, eager_new = make()
    for _ in range(12):
        short = pkg.kv_cache_reserve(eager_cache, eager_lens, eager_new)[1]
        slots = pkg.kv_slot_map(eager_cache, eager_lens, eager_new, 15)
        eager_lens.add_(eager_new)
        for graph, cache, lens, _, missing, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, cache, lens, _, missing, got in graphs:
            assert torch.equal(cache.page_table, eager_cache.page_table) and torch.equal(missing, short)
            assert all(torch.equal(a, b) for a, b in zip(got, slots))
