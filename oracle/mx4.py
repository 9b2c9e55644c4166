"""A paged cache held in 4 bits and its attention, in 64 bits on the CPU.

The format: each value a 4-bit float (sign, two exponent bits, one mantissa bit), each 32
dims of a row under a power of two 2^(byte - 127); byte 255 makes its block NaN.  Plain
restatements of the operators' definitions; none has a counterpart in the reference.
"""
from __future__ import annotations

import math

import torch

from . import paged

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
LARGEST = 1.5 * 2.0 ** 127


def steps(most: torch.Tensor) -> torch.Tensor:
    """The bytes of blocks whose largest magnitudes are ``most`` (fp64): the smallest e of
    -126 and up with most <= 7 x 2^e."""
    e = torch.where(most > 0, torch.frexp(most.clamp(max=LARGEST))[1], -122).clamp_min(-122) - 4
    for _ in range(2):
        e = torch.where(most.clamp(max=LARGEST) > 7 * torch.exp2(e.double()), e + 1, e)
    return torch.where(torch.isfinite(most), e.long() + 127, 255)


def round_to(x: torch.Tensor, step) -> torch.Tensor:
    """Codes 0 .. 15 of values x (fp64) under their steps: the nearest, ties to the even code."""
    far = ((x.abs() / step)[..., None] - GRID).abs()
    near = far == far.amin(-1, keepdim=True)
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])  # even codes first
    return torch.where(near, order, 9).argmin(-1) + torch.signbit(x).long() * 8


def stored(x: torch.Tensor) -> tuple:
    """x [..., hd] -> (codes [..., hd] 0 .. 15, bytes [..., hd / 32])."""
    x = x.double().unflatten(-1, (-1, 32))
    scales = steps(x.abs().amax(-1))  # (a NaN is the largest)
    step = torch.exp2(scales.double() - 127)[..., None]
    codes = torch.where(scales[..., None] < 255, round_to(x, step), 0)
    return codes.flatten(-2), scales


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 values of codes [..., hd] under bytes [..., hd / 32]."""
    x = GRID[codes & 7] * torch.where(codes > 7, -1.0, 1.0)
    step = torch.exp2(scales.double() - 127)
    step = torch.where(scales == 255, math.nan, step)
    return x * step.repeat_interleave(32, -1)


def pack(codes: torch.Tensor, scales: torch.Tensor) -> tuple:
    """The bytes of a cache: codes two a byte, the lower dim in the low bits."""
    return ((codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8), scales.to(torch.uint8))


def unpack(codes: torch.Tensor, scales: torch.Tensor) -> tuple:
    codes, scales = codes.view(torch.uint8).long(), scales.view(torch.uint8).long()
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2), scales


def attend(q, k, v, page_table, lengths, scale=None, window=0, softcap=0.0, slopes=None):
    """(out, spread) fp64 [B, T, Hq, hd]: token t of a sequence stands at lengths[b] - T + t;
    k, v [pages, Hkv, page, hd] fp64, the values of a cache."""
    B, T, Hq, hd = q.shape
    pages, Hkv, page, _ = k.shape
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(B, T, Hq, hd, dtype=torch.float64)
    spread = torch.zeros_like(out)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), page_table.shape[1] * page)
        if n == 0 or pages == 0:
            continue
        at = torch.arange(n)
        ids = page_table[b].long()[at // page]
        named = (ids >= 0) & (ids < pages)
        ids = ids.clamp(0, pages - 1)
        for t in range(T):
            end = n - (T - 1 - t)
            seen = named & (at < end)
            if window:
                seen &= at >= end - window
            for h in range(Hq):
                g = h // (Hq // Hkv)
                bias = None if slopes is None else slopes[h].double() * (end - 1 - at)
                out[b, t, h], spread[b, t, h] = paged.attend(
                    q[b, t, h], k[ids, g, at % page], v[ids, g, at % page], seen, scale, softcap,
                    bias)
    return out, spread
