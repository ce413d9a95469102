"""The serving operators (rotary positions, a paged int8 cache, attention over it) restated in plain tensor code, on any device.
TEST INFRASTRUCTURE ONLY, like the rest of this directory.

Values are computed in 64 bits from the definitions; what the operators define by fp32 operations (codes and scales: whole numbers and
their units) by those operations, one elementary tensor operation each.
"""
from __future__ import annotations

import math

import torch


def turn(x, cs, interleaved, inverse=False):
    """x [..., D] rotated by cs [..., rot/2, 2] in x's own type, one operation at a time."""
    half = cs.shape[-2]
    c, s = cs[..., 0], -cs[..., 1] if inverse else cs[..., 1]
    y = x.clone()
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., i], x[..., j]
    y[..., i] = a * c - b * s
    y[..., j] = b * c + a * s
    return y


def scale_of(most):
    return most / torch.full((), 127.0, dtype=most.dtype, device=most.device)


def codes(x, scale):
    ok = (scale > 0) & torch.isfinite(scale)
    return torch.where(ok, (x / scale).round().clamp(-127, 127), torch.zeros_like(x)).to(torch.int8)


def absmax(x):
    """Largest magnitude over the last axis, NaN if there is one."""
    return x.abs().amax(-1)


def append(k, v, kc, vc, ks, vs, table, lens, cu, q=None, cs=None, interleaved=False):
    """Like the operator, sequence by sequence, on copies: (kc, vc, ks, vs, q8, q_scale).  `cs`: the rotary table."""
    kc, vc, ks, vs = kc.clone(), vc.clone(), ks.clone(), vs.clone()
    page, block = kc.shape[2], kc.shape[2] // ks.shape[2]
    S = table.shape[0]
    cu = list(range(S + 1)) if cu is None else cu.tolist()
    q8 = qs = None
    if q is not None:
        q8, qs = torch.zeros(q.shape, dtype=torch.int8, device=q.device), torch.zeros(q.shape[:2], device=q.device)
    for s in range(S):
        n, length = cu[s + 1] - cu[s], int(lens[s])
        if n == 0 or length == 0:
            continue
        rows, first = slice(cu[s], cu[s + 1]), length - n
        pos = torch.arange(first, length, device=k.device)
        def spun(x):
            return x[rows].float() if cs is None else turn(x[rows].float(), cs[pos][:, None], interleaved)
        if q is not None:
            x = spun(q)
            qs[rows] = scale_of(absmax(x))
            q8[rows] = codes(x, qs[rows][..., None])
        for x, cache, scale in ((spun(k), kc, ks), (v[rows].float(), vc, vs)):
            for b in range(first // block, (length - 1) // block + 1):
                lo, hi = max(first, b * block), min(length, (b + 1) * block)
                pg, sl = int(table[s, lo // page]), lo % page
                blk, b0 = sl // block, sl // block * block
                new = scale_of(absmax(x[lo - first:hi - first].transpose(0, 1).flatten(1)))          # [heads]
                if lo > b * block:
                    old = scale[pg, :, blk].clone()
                    new = torch.where(old.isnan() | new.isnan(), torch.full_like(old, math.nan), torch.maximum(old, new))
                    ok = (new > 0) & torch.isfinite(new)
                    ratio = torch.where(ok, old / new, torch.zeros_like(new))
                    was = cache[pg, :, b0:sl]
                    moved = (new != old)[:, None, None]
                    cache[pg, :, b0:sl] = torch.where(moved, (was.float() * ratio[:, None, None]).round().to(torch.int8), was)
                scale[pg, :, blk] = new
                cache[pg, :, sl:sl + hi - lo] = codes(x[lo - first:hi - first].transpose(0, 1), new[:, None, None])
    return kc, vc, ks, vs, q8, qs


def gather(cache, scale, table_row, n):
    """The first n tokens of a sequence in 64 bits: [heads, n, D]."""
    page, block = cache.shape[2], cache.shape[2] // scale.shape[2]
    pages = table_row[:-(-n // page)].long()
    x = cache[pages].double() * scale[pages].double().repeat_interleave(block, -1)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def attention(q8, qs, kc, vc, ks, vs, table, lens, cu, causal, sm_scale):
    """(o, lse in the log2 domain, |o|'s bound sum p|v| / sum p, largest p|v|max / sum p) in 64 bits; rows of no sequence stay NaN."""
    T, H, D = q8.shape
    Hkv, S = kc.shape[1], table.shape[0]
    cu = list(range(S + 1)) if cu is None else cu.tolist()
    o = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q8.device)
    lse, big, top = (torch.full(s, math.nan, dtype=torch.float64, device=q8.device) for s in ((T, H), (T, H, D), (T, H)))
    for s in range(S):
        n, length = cu[s + 1] - cu[s], int(lens[s])
        rows = slice(cu[s], cu[s + 1])
        if n == 0:
            continue
        if length == 0:
            o[rows], lse[rows], big[rows], top[rows] = 0, -math.inf, 0, 0
            continue
        k, v = gather(kc, ks, table[s], length), gather(vc, vs, table[s], length)
        q = (q8[rows].double() * qs[rows].double()[..., None]).transpose(0, 1).reshape(Hkv, H // Hkv * n, D)
        x = (q @ k.transpose(1, 2) * sm_scale).view(H, n, length)
        if causal:
            seen = torch.arange(length, device=x.device)[None] <= torch.arange(length - n, length, device=x.device)[:, None]
            x = x.masked_fill(~seen, -math.inf)
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = p.sum(-1, keepdim=True)
        w = torch.where(l > 0, p / l, torch.zeros_like(p))
        w = torch.where(l.isnan(), l, w).view(Hkv, -1, length)
        o[rows] = (w @ v).view(H, n, D).transpose(0, 1)
        big[rows] = (w @ v.abs()).view(H, n, D).transpose(0, 1)
        top[rows] = (w * v.abs().amax(-1)[:, None]).amax(-1).view(H, n).T
        lse[rows] = ((m + l.log()) / math.log(2)).view(H, n).T
    return o, lse, big, top
