"""What page tables from lengths, attention under shared prefixes and sampling refuse before any GPU work."""
import ctypes
import importlib
import math

import pytest
import torch

P = 0x10000  # a fake, never-dereferenced, 16-byte aligned device address


@pytest.fixture(scope="module")
def L():
    return importlib.import_module("llm-inference-optimizer_amd._lib")


@pytest.fixture(scope="module")
def lib(L):
    return L.load()


def _cache(L, **kw):
    args = dict(k=P, v=P, k_scale=P, v_scale=P, page_table=P, table_stride=8, table_width=8, pages=10, kv_heads=2,
                page_size=16, head_dim=64, format=L.KV_INT8)
    args.update(kw)
    return ctypes.byref(L.KvCacheStruct(**args))


def _expect(lib, status, code, message):
    assert status == code
    assert message in lib.mi355_last_error().decode()


@pytest.mark.parametrize("kw,code,message", [
    (dict(dtype=0), -2, "fp16 or bf16"), (dict(tokens=129), -2, "tokens <= 128"), (dict(heads=3), -1, "multiple of kv_heads"),
    (dict(batch=1 << 18, tokens=64), -2, "limits"), (dict(q=0), -1, "null"), (dict(q=P + 8), -2, "aligned"),
    (dict(strides=[64, 64, 4]), -2, "multiples of 8"), (dict(strides=[64, -64, 64]), -1, "strides"),
    (dict(work=P + 8, bytes=64), -1, "workspace"), (dict(work=P, bytes=-1), -1, "workspace"),
    (dict(count=-1), -1, "group_count"), (dict(count=5), -1, "group_count"), (dict(prefix=0), -1, "null"),
    (dict(count=3), -1, "multiple of group_count"), (dict(cache=dict(k=0)), -1, "null"),
    (dict(cache=dict(page_size=24)), -2, "page_size"), (dict(cache=dict(k_scale=0)), -1, "scales")])
def test_shared_prefix_abi_rejects(L, lib, kw, code, message):
    a = dict(q=P, batch=4, tokens=2, heads=4, strides=[64] * 3, dtype=1, work=None, bytes=0, prefix=P, groups=None, count=2,
             cache={})
    a.update(kw)
    strides = (ctypes.c_int64 * 3)(*a["strides"])
    _expect(lib, lib.mi355_shared_prefix_attention_fwd(
        _cache(L, **a["cache"]), a["q"], P, P, None, a["prefix"], a["groups"], a["count"], None, 0, 0, a["batch"], a["tokens"],
        a["heads"], strides, 1.0, a["dtype"], a["work"], a["bytes"], None), code, message)


def test_shared_prefix_empty_is_noop(L, lib):
    strides = (ctypes.c_int64 * 3)(64, 64, 64)
    for batch, tokens, heads in ((0, 1, 4), (4, 0, 4), (4, 1, 0)):
        assert lib.mi355_shared_prefix_attention_fwd(_cache(L), 0, 0, 0, None, 0, None, 0, None, 0, 0, batch, tokens, heads,
                                                     strides, 1.0, 1, None, 0, None) == 0
    for args in ((0, 1, 4, 0), (4, 129, 4, 1), (4, 1, 3, 1), (4, 1, 4, 5), (4, 1, 4, -1)):
        assert lib.mi355_shared_prefix_attention_workspace(_cache(L), *args) == 0
    assert lib.mi355_shared_prefix_attention_workspace(None, 1, 1, 2, 1) == 0


@pytest.mark.parametrize("kw,code,message", [
    (dict(batch=-1), -1, "sizes"), (dict(stride=7), -1, "out_stride"), (dict(batch=1 << 24), -2, "limits"),
    (dict(cache=dict(pages=1 << 30)), -2, "limits"), (dict(batch=1 << 20, cache=dict(table_width=1 << 11, table_stride=1 << 11), stride=1 << 11), -2, "limits"),
    (dict(lens=0), -1, "null"), (dict(out=0), -1, "null"), (dict(missing=0), -1, "null"),
    (dict(out=P, stride=9), -1, "in place"), (dict(cache=dict(page_table=0), out=P + 64), -1, "null"),
    (dict(cache=dict(pages=0)), -1, "without pages"), (dict(cache=dict(pages=10 ** 6), work=None), -1, "workspace"),
    (dict(batch=2000, work=P + 4), -1, "workspace"), (dict(batch=5000, bytes=16), -1, "workspace"),
    (dict(cache=dict(page_size=20)), -2, "page_size")])
def test_reserve_abi_rejects(L, lib, kw, code, message):
    a = dict(lens=P, out=P + 4096, stride=8, missing=P, batch=3, work=P, bytes=1 << 30, cache={})
    a.update(kw)
    _expect(lib, lib.mi355_kv_cache_reserve_fwd(_cache(L, k=0, v=0, **a["cache"]), a["lens"], None, a["out"], a["stride"],
                                                a["missing"], a["batch"], a["work"], a["bytes"], None), code, message)


@pytest.mark.parametrize("kw,code,message", [
    (dict(batch=-1), -1, "sizes"), (dict(tokens=-1), -1, "sizes"), (dict(batch=1 << 24), -2, "limits"),
    (dict(tokens=1 << 31), -2, "limits"), (dict(batch=0), -1, "no sequence"), (dict(lens=0), -1, "null"),
    (dict(new=0), -1, "null"), (dict(slots=0), -1, "null"), (dict(cache=dict(page_table=0)), -1, "null"),
    (dict(cache=dict(table_width=0)), -1, "without pages"), (dict(batch=5000, work=P + 8), -1, "workspace")])
def test_slot_map_abi_rejects(L, lib, kw, code, message):
    a = dict(lens=P, new=P, slots=P, batch=3, tokens=5, work=P, bytes=1 << 20, cache={})
    a.update(kw)
    _expect(lib, lib.mi355_kv_slot_map_fwd(_cache(L, **a["cache"]), a["lens"], a["new"], a["slots"], P, P, a["batch"],
                                           a["tokens"], a["work"], a["bytes"], None), code, message)


def test_pages_abi_empty_is_noop(L, lib):
    assert lib.mi355_kv_cache_reserve_fwd(_cache(L), 0, 0, 0, 8, 0, 0, None, 0, None) == 0
    assert lib.mi355_kv_slot_map_fwd(_cache(L), 0, 0, 0, 0, 0, 3, 0, None, 0, None) == 0
    assert lib.mi355_kv_cache_reserve_workspace(_cache(L), 0) == 0 and lib.mi355_kv_cache_reserve_workspace(None, 3) == 0
    assert lib.mi355_kv_slot_map_workspace(0) == 0


@pytest.mark.parametrize("kw,code,message", [
    (dict(dtype=5), -1, "unknown dtype"), (dict(rows=-1), -1, "sizes"), (dict(vocab=0), -1, "sizes"),
    (dict(stride=99), -1, "sizes"), (dict(rows=1 << 20), -2, "limits"), (dict(vocab=1 << 20, stride=1 << 20), -2, "limits"),
    (dict(logits=0), -1, "null"), (dict(uniform=0), -1, "null"), (dict(tokens=0), -1, "null")])
def test_sample_abi_rejects(lib, kw, code, message):
    a = dict(logits=P, uniform=P, tokens=P, rows=2, vocab=100, stride=100, dtype=1)
    a.update(kw)
    _expect(lib, lib.mi355_sample_tokens_fwd(a["logits"], a["uniform"], a["tokens"], None, None, None, None, None, 1.0, 0, 1.0,
                                             0.0, a["rows"], a["vocab"], a["stride"], a["dtype"], P, 1 << 40, None), code,
            message)


def test_sample_abi_empty_is_noop(lib):
    assert lib.mi355_sample_tokens_fwd(0, 0, 0, None, None, None, None, None, 1.0, 0, 1.0, 0.0, 0, 100, 100, 1, None, 0,
                                       None) == 0
    assert lib.mi355_sample_tokens_workspace(0, 100) == 0 and lib.mi355_sample_tokens_workspace(1, 1 << 20) == 0


@pytest.mark.parametrize("kw", [dict(temperature=-0.1), dict(temperature=math.nan), dict(temperature="1"), dict(top_k=-1),
                                dict(top_k=1.5), dict(top_p=1.01), dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=2),
                                dict(min_p=None)])
def test_sample_refuses_settings(pkg, kw):
    with pytest.raises((ValueError, TypeError)):
        pkg.sample_tokens(torch.zeros(2, 5), torch.zeros(2), **kw)


def test_cpu_tensors_are_refused(pkg):
    with pytest.raises(AssertionError, match="GPU"):
        pkg.sample_tokens(torch.zeros(2, 5), torch.zeros(2))
    cache = pkg.KVCache(torch.zeros(2, 1, 16, 16).half(), torch.zeros(2, 1, 16, 16).half(), torch.zeros(1, 2, dtype=torch.int32))
    n = torch.ones(1, dtype=torch.int32)
    for call in (lambda: pkg.kv_cache_reserve(cache, n), lambda: pkg.kv_slot_map(cache, n, n, 1),
                 lambda: pkg.shared_prefix_attention(torch.zeros(1, 1, 1, 16).half(), cache, n, n)):
        with pytest.raises(AssertionError, match="GPU"):
            call()
