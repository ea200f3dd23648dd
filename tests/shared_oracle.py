"""64-bit forms, on the CPU, of attention under shared prefixes, of page tables and slot maps from lengths, and of drawing
tokens."""
from __future__ import annotations

import math

import torch
from kv_oracle import cpu


def members(batch, count, groups):
    """[(first, size)] of the groups; a boundary below an earlier one counts as that one."""
    if groups is None:
        return [(g * (batch // count), batch // count) for g in range(count)] if count else []
    at = []
    for g in groups:
        at.append(max([max(0, min(int(g), batch)), *at]))
    return [(at[g], at[g + 1] - at[g]) for g in range(count)]


def shared_slots(batch, lens, prefix, groups):
    """(first sequence of the group, shared slots) of each sequence."""
    out = [(b, 0) for b in range(batch)]
    for g, (first, size) in reversed(list(enumerate(members(batch, len(prefix), groups)))):
        for b in range(first, first + size):
            out[b] = (first, max(0, min(int(prefix[g]), int(lens[b]))))
    return out


def values(pools, table, page_size, b, first, last):
    """Keys and values [kv_heads, n, d] (64 bits) of slots first .. last - 1 of sequence b, and which have a place."""
    slot = torch.arange(first, last)
    page, place = table[b, slot // page_size].long(), slot % page_size
    there = (page >= 0) & (page < pools[0][0].shape[0])
    page = torch.where(there, page, 0)
    out = []
    for pool, scale in pools:
        x = pool[page, :, place].double()
        if scale is not None:
            x = x * scale[page, :, place].double()[..., None]
        out.append(torch.where(there[:, None, None], x, 0.0).transpose(0, 1))
    return out[0], out[1], there


def attention(q, cache, lens, prefix, groups=None, new=None, mask=None, scale=None):
    """(value, bound) of shared_prefix_attention's output; the bound is that of kv_oracle.attention, whose products,
    exponentials and sums are the same in another order."""
    batch, t, hq, d = q.shape
    q = cpu(q).double()
    kvh = cache.k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    cap = cache.page_table.shape[1] * cache.k.shape[2]
    lens = [max(0, min(int(n), cap)) for n in lens]
    table, page_size = cpu(cache.page_table), cache.k.shape[2]
    pools = [(cpu(pool.float()), cpu(scale)) for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    prefixes = {}
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, (first, shared) in enumerate(shared_slots(batch, lens, [int(p) for p in prefix], groups)):
        n, fresh = lens[b], t if new is None else max(0, min(int(new[b]), t))
        last = min(n + fresh, cap)
        if (first, shared) not in prefixes:
            prefixes[first, shared] = values(pools, table, page_size, first, 0, shared)
        k, v, there = (torch.cat(x, 1 if x[0].dim() == 3 else 0) for x in
                       zip(prefixes[first, shared], values(pools, table, page_size, b, shared, last)))
        for i in range(fresh):
            see = there.clone()
            drafted = torch.arange(t) <= i if mask is None else mask[b if mask.shape[0] > 1 else 0, i].cpu()
            see[n:last] &= drafted[:last - n]
            idx = see.nonzero()[:, 0]
            if not len(idx):
                continue
            for h in range(kvh):
                rows = slice(h * hq // kvh, (h + 1) * hq // kvh)
                kk, vv, qq = k[h][idx], v[h][idx], q[b, i, rows]
                p = torch.softmax(qq @ kk.T * scale, -1)
                e = (d + 8) * 2.0 ** -24 * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) * abs(scale)
                rel = 2 * (e + 2.0 ** -22 + len(idx) * 2.0 ** -24) + 2.0 ** -17 + 2.0 ** -22
                out[b, i, rows] = p @ vv
                bound[b, i, rows] = rel * (p @ vv.abs())
    return out, bound


def reserve(table, pages, page_size, lens, new=None):
    """(table, missing), entry by entry."""
    need = [-(-(max(0, a) + max(0, m)) // page_size) for a, m in zip(lens, new or [0] * len(lens))]
    named = [[p if 0 <= p < pages else -1 for p in row[:n]] for row, n in zip(table, need)]
    kept = {p for row in named for p in row}
    free = iter([p for p in range(pages) if p not in kept])
    out = [[p if p >= 0 else next(free, -1) for p in row] for row in named]
    missing = [n - sum(p >= 0 for p in row) for n, row in zip(need, out)]
    return [row + [-1] * (len(table[0]) - len(row)) for row in out], missing


def slot_map(table, pages, page_size, lens, new, tokens):
    out = []
    for b, (a, m) in enumerate(zip(lens, new)):
        for position in range(max(0, a), max(0, a) + max(0, m)):
            c = position // page_size
            page = table[b][c] if c < len(table[b]) else -1
            out.append((page * page_size + position % page_size if 0 <= page < pages else -1, b, position))
    return (out + [(-1, -1, 0)] * tokens)[:tokens]


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logarithm of its probability, least distance of a decision from its border) of one row x (1-d, CPU), from
    the definition.  Distances are relative to the weights' total: of u from the cumulated probabilities on its sides,
    and of the rank's mass from top_p."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    temperature, top_p, min_p, u = f32(temperature), f32(top_p), f32(min_p), f32(u)
    u = 0.0 if math.isnan(u) else min(max(u, 0.0), 1 - 2.0 ** -24)
    x = x.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.max()
    if top == -math.inf:
        return -1, -math.inf, 1.0
    order = torch.argsort(-x, stable=True)
    if not temperature > 0:
        return int(order[0]), 0.0, 1.0
    if top == math.inf:
        w = (x == top).double()
    else:
        w = torch.where(x == -math.inf, 0.0, torch.exp((x - top) / temperature))
    if 0 < top_k < len(x):
        order = order[:top_k]
    ranked = w[order]
    upto = torch.cumsum(ranked, 0)
    keep, near = torch.ones(len(order), dtype=torch.bool), 1.0
    if top_p < 1:
        # a mass exactly at the border (equal weights) is decided by the definition, not by rounding
        gap = ((upto - ranked) / upto[-1] - top_p)[1:]
        keep[1:] &= gap < 0
        near = min(near, float(gap.abs().min()) if len(gap) else 1.0)
    if min_p > 0:
        keep &= ranked >= min_p
        near = min(near, float((ranked - min_p).abs()[ranked != min_p].min()) if (ranked != min_p).any() else 1.0)
    keep[0] = True
    index, at = torch.sort(order[keep])
    ranked = ranked[keep][at]
    index, ranked = index[ranked > 0], ranked[ranked > 0]
    upto = torch.cumsum(ranked, 0)
    past = (upto > u * upto[-1]).nonzero()
    i = int(past[0]) if len(past) else len(index) - 1
    if len(upto) > 1 and u > 0:  # 0 is met exactly: the first token with any weight
        near = min(near, float((upto[:-1] / upto[-1] - u).abs().min()))
    return int(index[i]), math.log(float(ranked[i] / upto[-1])), near
