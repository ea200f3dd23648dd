"""64-bit forms of rotary positions, the quantised cache and attention over it, on the CPU, and what fp32 arithmetic
and the final rounding may differ from them by."""
from __future__ import annotations

import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def cpu(t):
    return None if t is None else t.detach().cpu()


def half_step(t, value):
    """Half a step of dtype t at |value| (64-bit): what one rounding may be off by, subnormals included."""
    tiny = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}[t]
    return value.abs() * torch.finfo(t).eps / 2 + tiny


def rotary(x, positions, inv_freq, scale=1.0, interleaved=False):
    """(value, bound without the final rounding) of x [batch, tokens, heads, d] in 64 bits.

    Bound: the angle's fraction of a turn is rounded to fp32 (2^-26 turns, 9.4e-8 radians), sine and cosine are at most
    2 ulp off (2^-23), and a product with scale, a product with x and the sum round once each (2^-24 each of at most
    scale (|x0| + |x1|)): 9.4e-8 + 1.2e-7 + 3 * 6e-8 = 4e-7 of scale (|x0| + |x1|)."""
    x = x.double()
    a = positions.double()[..., None] * inv_freq.double()
    c, s = (a.cos() * scale)[:, :, None], (a.sin() * scale)[:, :, None]
    n = inv_freq.numel()
    idx = torch.arange(n)
    i0, i1 = (2 * idx, 2 * idx + 1) if interleaved else (idx, idx + n)
    y, bound = x.clone(), torch.zeros_like(x)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    b = 4e-7 * abs(scale) * (x0.abs() + x1.abs())
    bound[..., i0], bound[..., i1] = b, b
    return y, bound


def encode(x, kind):
    """Codes and scales of fp32 rows [..., d], by the formula in fp32 (IEEE division, ties to even)."""
    s = (x.abs().amax(-1) / TOP[kind]).clamp(min=1e-8)
    y = x / s[..., None]
    return (y.round().clamp(-127, 127).to(torch.int8) if kind == torch.int8 else y.to(kind)), s


def place(cache, b, slot):
    """(page, place) of a slot, or None."""
    table, page_size = cpu(cache.page_table), cache.k.shape[2]
    if not 0 <= slot < table.shape[1] * page_size:
        return None
    page = int(table[b, slot // page_size])
    return (page, slot % page_size) if 0 <= page < cache.k.shape[0] else None


def values(cache, b, first, last):
    """Keys and values [kv_heads, n, d] (64 bits) of slots first .. last - 1 of sequence b, and which have a place."""
    k, v, ks, vs = cpu(cache.k), cpu(cache.v), cpu(cache.k_scale), cpu(cache.v_scale)
    h, d, n = k.shape[1], k.shape[3], last - first
    out, there = torch.zeros((2, h, n, d), dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        at = place(cache, b, first + i)
        if at is None:
            continue
        there[i] = True
        for side, (pool, scale) in enumerate(((k, ks), (v, vs))):
            out[side, :, i] = pool[at[0], :, at[1]].double() if scale is None else \
                pool[at[0], :, at[1]].float().double() * scale[at[0], :, at[1], None].double()
    return out[0], out[1], there


def attention(q, cache, lens, new=None, mask=None, scale=None):
    """(value, bound) of tree_attention's output [batch, tokens, q_heads, d].

    Bound, for a row with weights p (sum 1) and A = sum p |v|: a score is an fp32 sum of d products (each exact in
    fp32 but for its rounding), multiplied by two fp32 factors and log2 e, so it is off by at most e = (d + 8) 2^-24
    sum |q k| scale; the exponential is off by 2^-22 + e relatively, the weight goes to the product with v in two
    16-bit parts (2^-17), the sums of n terms round by n 2^-24 at most in any order, and numerator and denominator each
    carry it: 2 (e + 2^-22 + n 2^-24) + 2^-17 + 2^-22 times A; then the final rounding."""
    batch, t, hq, d = q.shape
    q = cpu(q).double()
    kvh = cache.k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    cap = cache.page_table.shape[1] * cache.k.shape[2]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        n, fresh = max(0, min(int(lens[b]), cap)), t if new is None else max(0, min(int(new[b]), t))
        last = min(n + fresh, cap)
        k, v, there = values(cache, b, 0, last)
        for i in range(fresh):
            see = there.clone()
            for s in range(n, last):
                j = s - n
                see[s] &= bool(mask[b if mask.shape[0] > 1 else 0, i, j]) if mask is not None else j <= i
            idx = see.nonzero()[:, 0]
            if not len(idx):
                continue
            for h in range(hq):
                kk, vv = k[h * kvh // hq][idx], v[h * kvh // hq][idx]
                s = kk @ q[b, i, h] * scale
                p = torch.softmax(s, 0)
                e = (d + 8) * 2.0 ** -24 * float((kk.abs() @ q[b, i, h].abs()).max()) * abs(scale)
                rel = 2 * (e + 2.0 ** -22 + len(idx) * 2.0 ** -24) + 2.0 ** -17 + 2.0 ** -22
                out[b, i, h] = p @ vv
                bound[b, i, h] = rel * (p @ vv.abs())
    return out, bound


def close(got, value, bound):
    """Asserts |got - value| <= bound + one rounding, element by element (NaN where the value is)."""
    g = cpu(got)
    err, allowed = (g.double() - value).abs(), bound + half_step(g.dtype, value) * (1 + 1e-6)
    nan = value.isnan()
    assert torch.equal(g.isnan(), nan), "NaN in other places"
    worst = ((err - allowed)[~nan]).max().item() if (~nan).any() else 0.0
    assert worst <= 0, f"off by {worst:.3g} beyond the bound (max error {err[~nan].max().item():.3g})"


def make_cache(pkg, kind, dtype, shape, table, seed, device="cuda"):
    """A cache of random entries: kind "16bit", "int8" or "e4m3", shape [pages, heads, page_size, d]."""
    g = torch.Generator().manual_seed(seed)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if kind == "16bit":
            pools.append(x.to(dtype).to(device))
            scales.append(None)
        else:
            c, s = encode(x, pkg.KV_FORMATS[kind])
            pools.append(c.to(device))
            scales.append(s.to(device))
    return pkg.KVCache(*pools, torch.as_tensor(table, dtype=torch.int32).to(device), *scales)


def shuffled_table(batch, per, spare, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(batch * per + spare, generator=g)[:batch * per].view(batch, per), batch * per + spare


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def random_tree(batch, tokens, seed):
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros((batch, tokens, tokens), dtype=torch.bool)
    for b in range(batch):
        for i in range(tokens):
            if i:
                mask[b, i] = mask[b, int(torch.randint(max(0, i - 5), i, (1,), generator=g))]
            mask[b, i, i] = True
    return mask
