"""Plain forms of the 4-bit cache operators, for the tests: dim by dim from the layout, in 64 bits."""

from __future__ import annotations

import math

import torch

GROUP = 32


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes [..., dim] int64, scales, offsets [..., dim / 32] in x's dtype) of 16-bit rows, every step in 64 bits."""
    dtype = x.dtype
    g = x.double().unflatten(-1, (-1, GROUP))
    sound = torch.isfinite(g).all(-1)
    z = torch.where(sound[..., None], g, torch.zeros_like(g))
    low, high = z.amin(-1), z.amax(-1)
    sound &= (high - low) <= torch.finfo(torch.float32).max
    low, high = torch.where(sound, low, 0.0), torch.where(sound, high, 0.0)
    scale = ((high - low) / 15).to(dtype)
    over = ~torch.isfinite((15 * scale.double() + low).to(dtype))
    scale = torch.where(over, (scale.view(torch.int16) - 1).view(dtype), scale)
    s = scale.double()[..., None]
    code = torch.where(s > 0, ((z - low[..., None]) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    code = torch.where(sound[..., None], code, 0.0)
    offset = torch.where(sound, low, math.nan).to(dtype)
    return code.long().flatten(-2), torch.where(sound, scale, torch.zeros_like(scale)), offset


def values(codes: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    s, o = (y.double().repeat_interleave(GROUP, -1) for y in (scales, offsets))
    return (codes.double() * s + o).to(scales.dtype)


def put(data: torch.Tensor, slot: int, part: int, codes, scales, offsets) -> None:
    """A token's codes [heads, dim] and pairs [heads, dim / 32] into pages [pages, heads, page / 8, 10 dim] (part 0: keys, 1: values)."""
    pages, heads, blocks, size = data.shape
    dim = size // 10
    page, off = divmod(slot, 8 * blocks)
    block, r = divmod(off, 8)
    run = data[page, :, block, part * 5 * dim:(part + 1) * 5 * dim]
    words = torch.zeros(heads, dim // 8, dtype=torch.int64, device=data.device)
    for d in range(dim):
        words[:, d // 8] |= codes[:, d] << (4 * (d % 8 // 2) + 16 * (d % 2))
    if dim == 128 and r in (2, 3, 6, 7):
        words = words.roll(8, -1)
    half = dim // 2
    for w in range(dim // 8):
        for b in range(4):
            run[:, r * half + 4 * w + b] = ((words[:, w] >> (8 * b)) & 255).to(torch.uint8)
    pairs = torch.stack([scales, offsets], -1).flatten(-2).contiguous().view(torch.uint8)
    run[:, 8 * half + r * dim // 8: 8 * half + (r + 1) * dim // 8] = pairs


def decoded(data: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Values [2, pages * page_size, heads, dim] of pages [pages, heads, page / 8, 10 dim], in dtype."""
    pages, heads, blocks, size = data.shape
    dim = size // 10
    parts = data.reshape(pages, heads, blocks, 2, 5 * dim)
    words = parts[..., : 4 * dim].contiguous().view(torch.int32).view(pages, heads, blocks, 2, 8, dim // 8)
    pairs = parts[..., 4 * dim:].contiguous().view(dtype).view(pages, heads, blocks, 2, 8, dim // GROUP, 2)
    codes = torch.empty(pages, heads, blocks, 2, 8, dim, dtype=torch.int64, device=data.device)
    for r in range(8):
        for d in range(dim):
            w = d // 8
            if dim == 128 and r in (2, 3, 6, 7):
                w = (w + 8) % 16
            codes[..., r, d] = (words[..., r, w] >> (4 * (d % 8 // 2) + 16 * (d % 2))) & 15
    x = values(codes, pairs[..., 0], pairs[..., 1])
    return x.permute(3, 0, 2, 4, 1, 5).reshape(2, pages * blocks * 8, heads, dim)


def evict(weights: list[float], keep: int, sinks: int, recent: int) -> list[int]:
    """Places that stay of one request's head, in order."""
    t = len(weights)
    if t <= keep:
        return list(range(t))
    middle = range(sinks, t - recent)
    best = sorted(middle, key=lambda i: (0 if math.isnan(weights[i]) else 1, -weights[i] if not math.isnan(weights[i]) else 0.0, i))
    return sorted([*range(sinks), *best[: keep - sinks - recent], *range(t - recent, t)])
