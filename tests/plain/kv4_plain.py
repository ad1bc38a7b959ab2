"""The 4-bit cache in 64 bits, element by element as its definition reads: groups of 32, m = bf16(min), s = bf16(range / 15),
code = rint((y - m) / s) within 0 .. 15, value m + s * code."""
import math

import torch

GROUP = 32


def _bf16(x):
    return x.to(torch.float32).to(torch.bfloat16)


def coded(y):
    """[..., dim] in 64 bits -> (codes uint8 [..., dim], pairs bfloat16 [..., groups, 2] = (s, m))."""
    y = y.double().unflatten(-1, (-1, GROUP))
    low, high = y.amin(-1), y.amax(-1)
    m, s = _bf16(low), _bf16((high - low) / 15.0)
    good = torch.isfinite(y).all(-1) & torch.isfinite(m) & torch.isfinite(s)
    step = torch.where(s == 0, torch.ones_like(s), s).double()[..., None]
    code = ((y - m.double()[..., None]) / step).round().clamp(0, 15)
    code = torch.where((good & (s != 0))[..., None], code, torch.zeros_like(code))
    nan = torch.full_like(s, math.nan)
    pairs = torch.stack((torch.where(good, s, nan), torch.where(good, m, nan)), -1)
    return code.flatten(-2).to(torch.uint8), pairs


def values(codes, pairs):
    """float64 [..., dim]."""
    s, m = pairs[..., 0].double(), pairs[..., 1].double()
    return (m[..., None] + s[..., None] * codes.unflatten(-1, (-1, GROUP)).double()).flatten(-2)


def put(pages, page, plane, head, slot, codes, pairs):
    """One row's codes [dim] and pairs [groups, 2] into pages uint8 [pages, 2, heads, runs, bytes] (CPU)."""
    groups = len(pairs)
    run = pages[page, plane, head, slot // 8]
    packed = codes[0::2] | codes[1::2] << 4
    bits = pairs.contiguous().view(torch.uint8).view(groups, 4)
    for g in range(groups):
        run[g * 128 + slot % 8 * 16:][:16] = packed[16 * g:16 * g + 16]
        run[128 * groups + slot % 8 * 4 * groups + 4 * g:][:4] = bits[g]


def get(pages, page, plane, head, slot):
    """(codes [dim], pairs [groups, 2]) of one row."""
    run = pages[page, plane, head, slot // 8]
    groups = len(run) // 160
    codes = torch.stack([run[g * 128 + slot % 8 * 16:][:16] for g in range(groups)])
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten()
    begin = 128 * groups + slot % 8 * 4 * groups
    return codes, run[begin:begin + 4 * groups].clone().view(torch.bfloat16).view(groups, 2)


def build(keys, held_values, lens, page_size, *, seed=0, spare=3, poison=255):
    """Pages and a block table of requests whose rows are keys[i], held_values[i] [length, heads, dim]: (pages, table, the float64 values
    that are held, [(keys, values)]).  Every byte that no row owns is ``poison`` (255: pairs of NaN)."""
    heads, dim = keys[0].shape[1:]
    needed = [-(-n // page_size) for n in lens]
    generator = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(needed) + spare, generator=generator)
    pages = torch.full((sum(needed) + spare, 2, heads, page_size // 8, 5 * dim), poison, dtype=torch.uint8)
    table = torch.full((len(lens), max(needed) + 2), -1, dtype=torch.int32)
    held, begin = [], 0
    for i, n in enumerate(lens):
        table[i, :needed[i]] = order[begin:begin + needed[i]].int()
        begin += needed[i]
        both = []
        for plane, rows in enumerate((keys[i], held_values[i])):
            codes, pairs = coded(rows)
            at = torch.arange(n)
            where, run, slot = table[i].long()[at // page_size], at % page_size // 8, at % 8
            groups = dim // GROUP
            packed = (codes[..., 0::2] | codes[..., 1::2] << 4).view(n, heads, groups, 16)
            bits = pairs.reshape(n, heads, groups * 2).view(torch.uint8).view(n, heads, groups * 4)
            for head in range(heads):
                flat = pages[:, plane, head]
                byte = torch.arange(16)
                for g in range(groups):
                    flat[where[:, None], run[:, None], g * 128 + slot[:, None] * 16 + byte] = packed[:, head, g]
                flat[where[:, None], run[:, None], 128 * groups + slot[:, None] * 4 * groups + torch.arange(4 * groups)] = bits[:, head]
            both.append(values(codes, pairs))
        held.append(tuple(both))
    return pages, table, held


def attention(q, keys, held_values, positions, scale, window=0):
    """float64: q [n, query heads, dim] at ``positions`` over keys, values [length, kv heads, dim] in 64 bits: (out [n, query heads, dim],
    sum of p |v| of the same shape: what a relative rounding of p is multiplied by)."""
    q, keys, held_values = q.double(), keys.double(), held_values.double()
    n, heads, dim = q.shape
    share = heads // keys.shape[1]
    keys, held_values = (t.repeat_interleave(share, dim=1) for t in (keys, held_values))
    scores = torch.einsum("nhd,thd->hnt", q, keys) * scale
    at = torch.arange(len(keys))[None, :]
    seen = at <= positions[:, None]
    if window:
        seen &= at > positions[:, None] - window
    scores = scores.masked_fill(~seen[None], -math.inf)
    p = scores.softmax(-1)
    p = torch.where(seen[None], p, torch.zeros_like(p))
    clean = torch.where(seen.any(0)[:, None, None], held_values, torch.zeros_like(held_values))
    return torch.einsum("hnt,thd->nhd", p, clean), torch.einsum("hnt,thd->nhd", p, clean.abs())


def turned(x, angles, rot, layout, gain=1.0, table=None):
    """x [n, heads, dim] in 64 bits, its first ``rot`` dimensions turned by angles [n, rot / 2] (or cosines and sines of ``table`` [n, rot])."""
    cosine, sine = (gain * angles.cos(), gain * angles.sin()) if table is None else (table[:, :rot // 2], table[:, rot // 2:])
    cosine, sine = cosine.double()[:, None], sine.double()[:, None]
    out = x.double().clone()
    if layout == 1:
        u, v = x[..., 0:rot:2].double(), x[..., 1:rot:2].double()
        out[..., 0:rot:2], out[..., 1:rot:2] = u * cosine - v * sine, v * cosine + u * sine
    else:
        u, v = x[..., :rot // 2].double(), x[..., rot // 2:rot].double()
        out[..., :rot // 2], out[..., rot // 2:rot] = u * cosine - v * sine, v * cosine + u * sine
    return out


def normed(x, weight, eps):
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return x if weight is None else x * weight.double()
