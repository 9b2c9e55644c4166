"""Full-length attention over rotated rows and a paged cache, in 64 bits on the CPU.

Plain restatements of the operators' definitions; none has a counterpart in the
reference, whose attention is banded and unrotated.  Every function returns, beside
the result, what its tests need to bound a kernel's rounding.
"""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def norm_rope(x, positions, inv_freq=None, weight=None, eps=1e-6, interleaved=False):
    """x [N, H, hd] -> fp64 [N, H, hd]: per-head RMSNorm (weight [hd] given), then the
    pairs of the first 2 len(inv_freq) dims rotated by positions * inv_freq."""
    y = x.double().clone()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    if inv_freq is None or inv_freq.numel() == 0:
        return y
    half = inv_freq.numel()
    out = y.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        t = positions.double() * inv_freq[i].double()
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def slots(page_table, rows, positions, page, pages):
    """(page, slot) of each token, or None where it has none."""
    B, width = page_table.shape
    found = []
    for n, p in enumerate(positions.tolist()):
        r = n if rows is None else int(rows[n])
        ok = p >= 0 and 0 <= r < B and p // page < width
        g = int(page_table[r, p // page]) if ok else -1
        found.append((g, p % page) if ok and 0 <= g < pages else None)
    return found


def attend(q, k, v, seen, scale, softcap=0.0, bias=None):
    """One query q [hd] over k, v [n, hd] where seen [n]; bias [n] is subtracted.
    Returns (out [hd], spread [hd]): spread = sum_j w_j |v_j - out|."""
    if not bool(seen.any()):
        z = torch.zeros(v.shape[1], dtype=torch.float64)
        return z, z
    q, k, v = q.double(), k.double()[seen], v.double()[seen]
    z = scale * (k @ q)
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    if bias is not None:
        z = z - bias.double()[seen]
    w = torch.softmax(z, 0)
    out = w @ v
    return out, w @ (v - out).abs()


def paged_decode(q, k_cache, v_cache, page_table, lengths, scale=None, window=0, softcap=0.0,
                 slopes=None, k_scale=1.0, v_scale=1.0):
    """(out, spread) fp64 [B, Hq, hd] of one query per sequence over a paged cache."""
    B, Hq, hd = q.shape
    pages, Hkv, page, _ = k_cache.shape
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(B, Hq, hd, dtype=torch.float64)
    spread = torch.zeros_like(out)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), page_table.shape[1] * page)
        if n == 0 or pages == 0:
            continue
        at = torch.arange(n)
        ids = page_table[b].long()[at // page]
        named = (ids >= 0) & (ids < pages)
        seen = named & (at >= n - window if window else torch.ones_like(named))
        ids = ids.clamp(0, pages - 1)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            k = k_cache[ids, g, at % page].float().double() * k_scale
            v = v_cache[ids, g, at % page].float().double() * v_scale
            bias = None if slopes is None else slopes[h].double() * (n - 1 - at)
            out[b, h], spread[b, h] = attend(q[b, h], k, v, seen, scale, softcap, bias)
    return out, spread


def packed_prefill(q, k, v, cu_seqlens, scale=None, window=0, softcap=0.0, slopes=None,
                   prefix=None):
    """(out, spread) fp64 [N, Hq, hd] of packed documents; rows of no document stay NaN."""
    N, Hq, hd = q.shape
    Hkv = k.shape[1]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.full((N, Hq, hd), math.nan, dtype=torch.float64)
    spread = torch.zeros_like(out)
    cu = [min(max(int(c), 0), N) for c in cu_seqlens]
    for d, (a, e) in enumerate(zip(cu, cu[1:])):
        p = 0 if prefix is None else int(prefix[d])
        j = torch.arange(max(0, e - a))
        for i in range(a, e, 32):
            t = torch.arange(i, min(i + 32, e))[:, None] - a
            seen = (j <= t) | (j < p)
            if window:
                seen &= t - j < window
            for h in range(Hq):
                g = h // (Hq // Hkv)
                x, y = k[a:e, g].double(), v[a:e, g].double()
                z = scale * (q[i:i + len(t), h].double() @ x.T)
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                if slopes is not None:
                    z = z - slopes[h].double() * (t - j).abs()
                w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                o = w @ y
                out[i:i + len(t), h] = o
                spread[i:i + len(t), h] = torch.einsum("nj,njd->nd", w,
                                                       (y - o[:, None]).abs())
    return out, spread
