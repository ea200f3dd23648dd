"""Calls of sample_tokens and shared_prefix_attention at the ends of what they allow: rows and groups beyond one launch's
share, the largest vocabulary, logits that hardly differ, settings at the ends of 32 bits, no workspace.  Bounds are those
of test_sampling.py and kv_oracle.attention."""
import ctypes
import importlib
import math

import pytest
import torch
from kv_oracle import close, ints
from shared_oracle import attention
from test_sampling import TYPES, _check, _logits
from test_shared_prefix import BF16, F16, _setup

pytestmark = pytest.mark.gpu


def test_more_rows_than_the_workspace_holds(pkg, cuda):
    """1100 rows, every one with settings of its own: rows are taken 1024 at a time."""
    x, u = _logits(1100, 300, torch.float16, 3)
    g = torch.Generator().manual_seed(5)
    pick = lambda values: torch.tensor(values)[torch.randint(len(values), (1100,), generator=g)]  # noqa: E731
    _check(pkg, cuda, x, u, temperature=pick([0.0, 0.7, 1.3]), top_k=pick([0, 1, 9, 100]).int(), top_p=pick([1.0, 0.9, 0.4]),
           min_p=pick([0.0, 0.1]))
    tokens = pkg.sample_tokens(x.to(cuda), u.to(cuda))
    assert torch.equal(tokens[1024:], pkg.sample_tokens(x[1024:].to(cuda), u[1024:].to(cuda)))


@pytest.mark.parametrize("rows,vocab", [(32768 + 5, 40), (2 * 128 + 3, 2 ** 20 - 8)])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=9, top_p=0.9)], ids=str)
def test_rows_beyond_one_pass(pkg, cuda, rows, vocab, settings):
    """More 4096ths of rows than 32768: rows are taken in turns, and draw what they draw alone."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn((rows, vocab), generator=g, device=cuda) * 3).half()
    u = torch.rand((rows,), generator=g, device=cuda)
    tokens = pkg.sample_tokens(x, u, **settings)
    for first, last in ((0, 100), (100, 129), (rows // 2, rows // 2 + 9), (rows - 9, rows)):
        assert torch.equal(tokens[first:last], pkg.sample_tokens(x[first:last], u[first:last], **settings))
    at = [0, 127, 128, rows - 6, rows - 1]
    _check(pkg, cuda, x[at].cpu(), u[at].cpu(), **settings)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [2 ** 20 - 1, 2 ** 20 - 16])
def test_the_largest_vocabulary(pkg, cuda, kind, vocab):
    x, u = _logits(2, vocab, TYPES[kind], 29, likely=60)
    for settings in (dict(), dict(top_p=0.9), dict(temperature=0.8, top_k=40), dict(temperature=0.0)):
        _check(pkg, cuda, x, u, **settings)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("settings", [dict(top_k=2000, top_p=0.7), dict(top_k=700, min_p=0.001), dict(top_k=4000, top_p=0.95, min_p=1e-4),
                                      dict(top_k=256, top_p=0.5), dict(top_p=0.99, min_p=1e-5)], ids=str)
def test_a_threshold_after_another(pkg, cuda, kind, settings):
    """Limits of many tokens, whose bins are looked for one after the other, or again."""
    for scale in (0.5, 2.0):
        x, u = _logits(5, 50000, TYPES[kind], 37, scale=scale, likely=30)
        _check(pkg, cuda, x, u, **settings)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.7), dict(top_k=10000), dict(min_p=0.5), dict(top_k=30000, top_p=0.3, min_p=0.9),
                                      dict(temperature=math.inf, top_p=0.7)], ids=str)
def test_logits_that_hardly_differ(pkg, cuda, kind, settings):
    """More tokens in one bin than a row's workgroup lists: equal logits, and ones within a thousandth."""
    u = torch.rand((3,), generator=torch.Generator().manual_seed(41))
    x = torch.full((3, 40001), 1.5)
    x[1] += torch.rand((40001,), generator=torch.Generator().manual_seed(43)) * 1e-3
    x[2, ::7] = -math.inf
    _check(pkg, cuda, x.to(TYPES[kind]), u, **settings)


@pytest.mark.parametrize("temperature", [1e-45, 1e-38, 1e-20, 1e20, 3e38])
def test_temperatures_at_the_ends(pkg, cuda, temperature):
    for dtype in (torch.float32, torch.bfloat16):
        x, u = _logits(4, 5000, dtype, 47)
        x[1] = 0.0
        x[2, 10] = x[2, 4000] = 40.0
        for settings in (dict(), dict(top_k=6), dict(top_p=0.5), dict(min_p=0.3)):
            _check(pkg, cuda, x, u, temperature=temperature, **settings)


def test_settings_of_any_stride(pkg, cuda):
    """Columns of a wider table, and one value for all rows by stride 0, give what packed ones give."""
    x, u = (t.to(cuda) for t in _logits(9, 1000, torch.float16, 53))
    table = torch.rand((9, 3), generator=torch.Generator().manual_seed(59)).to(cuda)
    want = pkg.sample_tokens(x, u, top_p=table[:, 1].contiguous(), min_p=(0.1 * table[:, 2]).contiguous())
    assert torch.equal(pkg.sample_tokens(x, u, top_p=table[:, 1], min_p=(0.1 * table)[:, 2]), want)
    k = torch.tensor([5], dtype=torch.int32, device=cuda)
    assert torch.equal(pkg.sample_tokens(x, u, top_k=k.expand(9)), pkg.sample_tokens(x, u, top_k=5))


@pytest.mark.parametrize("kind,dtype", [("16bit", F16), ("16bit", BF16), ("int8", F16), ("e4m3", BF16)])
def test_attention_without_a_workspace(pkg, cuda, kind, dtype):
    """The C entry computes the same, row by row, when it is given no workspace."""
    L = importlib.import_module("llm-inference-optimizer_amd._lib")
    lib = L.load()
    cache, q, lens, starts = _setup(pkg, kind, dtype, (6, 2, 96), [4, 3], [150, 37], [9, 0, 30, 70, 5, 16, 1], 3, 32, 61)
    c = L.KvCacheStruct(k=cache.k.data_ptr(), v=cache.v.data_ptr(), k_scale=cache.k_scale.data_ptr() if kind != "16bit" else 0,
                        v_scale=cache.v_scale.data_ptr() if kind != "16bit" else 0, page_table=cache.page_table.data_ptr(),
                        table_stride=cache.page_table.stride(0), table_width=cache.page_table.shape[1], pages=cache.k.shape[0],
                        kv_heads=2, page_size=32, head_dim=96,
                        format={"16bit": L.KV_16BIT, "int8": L.KV_INT8, "e4m3": L.KV_E4M3}[kind])
    out = torch.empty_like(q)
    given = [ints(lens), ints([150, 37]), ints(starts)]
    strides = (ctypes.c_int64 * 3)(*q.stride()[:3])
    code = lib.mi355_shared_prefix_attention_fwd(
        ctypes.byref(c), q.data_ptr(), out.data_ptr(), given[0].data_ptr(), None, given[1].data_ptr(), given[2].data_ptr(), 2,
        None, 0, 0, 7, 3, 6, strides, 96 ** -0.5, 1 if dtype == F16 else 2, None, 0,
        torch.cuda.current_stream().cuda_stream)
    assert code == 0, lib.mi355_last_error().decode()
    close(out, *attention(q, cache, lens, [150, 37], starts))


def test_more_groups_than_threads(pkg, cuda):
    """1050 groups of one or two sequences."""
    sizes = [1 + i % 2 for i in range(1050)]
    prefix, own = [1 + (13 * i) % 40 for i in range(1050)], [(7 * i) % 11 for i in range(sum(sizes))]
    cache, q, lens, starts = _setup(pkg, "int8", F16, (2, 1, 64), sizes, prefix, own, 1, 16, 67)
    out = pkg.shared_prefix_attention(q, cache, ints(lens), ints(prefix), ints(starts))
    close(out, *attention(q, cache, lens, prefix, starts))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("settings", [dict(top_k=360), dict(top_k=400, temperature=0.7), dict(top_p=0.5), dict(top_p=0.6, temperature=2.0),
                                      dict(min_p=0.58), dict(top_k=900, top_p=0.55)], ids=str)
def test_thresholds_right_below_zeros(pkg, cuda, kind, settings):
    """Bins of logits end at 0: zeros of both signs belong to the one above."""
    g = torch.Generator().manual_seed(73)
    x = torch.full((4, 3000), -3.0)
    x[:, :300] = 0.0
    x[:, 300:400] = -0.0
    x[:, 400:900] = -0.002 - 0.1 * torch.rand((4, 500), generator=g)
    x[:, 900:910] = 0.5
    x = x[:, torch.randperm(3000, generator=g)]
    _check(pkg, cuda, x.to(TYPES[kind]), torch.rand((4,), generator=g), **settings)
