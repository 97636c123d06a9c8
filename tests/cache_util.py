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


def visible(n: int, t: int, bits: torch.Tensor | None, window: int, sinks: int) -> torch.Tensor:
    """[n, t + n]: what the n nodes behind t cached tokens see. bits: their own tree's [n, n], None for a chain; window 0: none."""
    i = torch.arange(n)
    if bits is None:
        tree = i[None] <= i[:, None]
        if window:
            tree &= i[None] > i[:, None] - window
    else:
        tree = bits.cpu()
    see = torch.ones(n, t + n, dtype=torch.bool)
    see[:, t:] = tree
    if window:
        for r in range(n):
            see[r, min(sinks, t): max(min(sinks, t), t - max(0, window - int(tree[r].sum())))] = False
    return see


def attention(q, k, v, data, dtype, tables, lengths, starts, bits, window=0, sinks=0, scale=None):
    """(out, lse, allowed error of out, of lse) in 64 bits, request by request, over the values that 4-bit pages stand for.

    bits: per request a bool [n, n] array of what a node sees, or None for a chain. The error that fp32 scores and sums with
    probabilities rounded to the inputs' type allow, with u = eps / 2 of that type:
      |out - ref| <= (u + 2 d) A + u |ref| + f,   A = sum_j w_j |v_j|  (w: exact weights)
    where u A is the rounding of the probabilities, u |ref| that of the result, and d bounds how far a score is off (in
    natural units): dim products summed in fp32, where the tensor cores may cut a sum instead of rounding it, are off by at most dim * 2^-23 * S
    with S = scale * sum |q||k|; the scaling, the shift by the maximum and exp2 by 2^-24 * 4 (|s| + |max| + 1) and by 2^-22 more. A
    weight then moves by about 2 d (its own score and the sum's). The products with the values are summed in fp32: 2^-23 a
    term and relative, as is the sum of the weights. fp16 probabilities below 2^-14 are off by up to 2^-25 (of a largest one of at least 2^7):
    f = 2^-32 sum_j |v_j| / l, and a result below 2^-14 is rounded by up to 2^-25 instead of u |ref|. The log of the sum is off
    by 2 d, the sum's rounding and 2^-22 (|lse| + 1).
    """
    total, heads, dim = q.shape
    kv = k.shape[1]
    page = 8 * data.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    held = decoded(data, dtype).double()
    out = torch.zeros(total, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((total, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b, t in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        if n == 0:
            continue
        place = torch.arange(t)
        slots = torch.tensor([int(tables[b][x // page]) * page + x % page for x in place.tolist()], dtype=torch.int64, device=q.device)
        see = visible(n, t, None if bits is None else bits[b], window, sinks).to(q.device)
        used = see.any(0)
        for g in range(kv):
            kk, vv = (torch.where(used[:, None], torch.cat([held[x][slots, g], y[lo:hi, g].double()]), 0.0) for x, y in ((0, k), (1, v)))
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                x = q[lo:hi, h].double()
                s = torch.where(see, (x @ kk.T) * scale, -math.inf)
                top = s.amax(-1, keepdim=True)
                top = torch.where(torch.isfinite(top), top, 0.0)
                e = torch.where(see, torch.exp(s - top), 0.0)
                l = e.sum(-1, keepdim=True)
                some = see.any(-1, keepdim=True)  # (a row that sees a key that is not finite is NaN, one that sees nothing 0)
                w = torch.where(some, e / l, torch.zeros_like(e))
                if bool(torch.isfinite(vv).all()):
                    o, a, f = w @ vv, w @ vv.abs(), see.double() @ vv.abs()
                else:  # a hidden value has no influence, not even as 0 * NaN
                    o, a, f = (torch.stack([y[i][see[i]] @ z[see[i]] for i in range(n)]) for y, z in ((w, vv), (w, vv.abs()), (see.double(), vv.abs())))
                out[lo:hi, h] = o
                lse[lo:hi, h] = torch.where(some, top + torch.log(l), -math.inf)[:, 0]
                big = torch.where(see, (x.abs() @ kk.abs().nan_to_num(0, 0, 0).T) * abs(scale), 0.0).amax(-1, keepdim=True).nan_to_num(0, 0, 0)
                d = 2.0 ** -23 * dim * big + 2.0 ** -24 * 4 * (2 * big + 1) + 2.0 ** -22
                sub = 2.0 ** -32 * f / l.clamp(min=1e-300) + 2.0 ** -25 if q.dtype == torch.float16 else 0.0
                tol[lo:hi, h] = (u + 2 * d + 2 * (t + n) * 2.0 ** -23) * a + u * o.abs() + sub
                lse_tol[lo:hi, h] = (2 * d + (t + n) * 2.0 ** -23)[:, 0] + 2.0 ** -22 * (lse[lo:hi, h].abs().nan_to_num(0, 0, 0) + 1)
    return out, lse, tol, lse_tol


def close(got, want, tol) -> bool:
    """Within the allowed error; NaN and infinities in the same places."""
    same = (got.double() == want) | (got.isnan() & want.isnan())
    return bool((same | ((got.double() - want).abs() <= tol)).all())


def weights(q, keys, slots, lengths, starts, lse, old, window=0, sinks=0, scale=None):
    """(sums, allowed error) in 64 bits of the attention that cached tokens are given. keys [slots, kv, dim], slots: per request.

    A term exp(s - lse) is off by a factor of e^d, d = dim * 2^-23 * S + 2^-24 * 4 (|s| + |lse| + 1) + 2^-22 (see attention),
    each addition by 2^-24 of what has been added up.
    """
    total, heads, dim = q.shape
    kv = keys.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, tol = old.double().clone(), torch.zeros(old.shape, dtype=torch.float64, device=q.device)
    for b, t in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        see = visible(hi - lo, t, None, window, sinks)[:, :t].to(q.device)
        for h in range(heads):
            g = h * kv // heads
            k = torch.where(see.any(0)[:, None], keys[slots[b], g].double(), 0.0)
            x = q[lo:hi, h].double()
            s = (x @ k.T) * scale
            y = lse[lo:hi, h, None].double()
            p = torch.where(see & (y != -math.inf), torch.exp(s - y), 0.0)
            d = dim * 2.0 ** -23 * (x.abs() @ k.abs().T) * abs(scale) + 2.0 ** -22 * (s.abs() + y.abs().nan_to_num(0, 0, 0) + 1) + 2.0 ** -22
            out[b, g, :t] += p.sum(0)
            tol[b, g, :t] += torch.where(p > 0, p * d.exp() * d, 0.0).sum(0)
    rows = (max((hi - lo for lo, hi in zip(starts, starts[1:])), default=0)) * heads // kv
    return out, tol + (rows + 2) * 2.0 ** -24 * out.abs()

