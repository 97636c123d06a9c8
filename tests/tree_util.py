"""Plain 64-bit forms of the tree verification operators, for the tests."""

from __future__ import annotations

import math

import numpy as np
import torch


def random_parents(n: int, rng: np.random.Generator, chain: float = 0.3) -> list[int]:
    """A random forest in which every parent comes before its children."""
    out = []
    for i in range(n):
        r = rng.random()
        out.append(-1 if i == 0 or r < 0.1 else i - 1 if r < 0.1 + chain else int(rng.integers(0, i)))
    return out


def ancestors(parents: list[int]) -> list[list[int]]:
    """Every node's path from its top down to itself."""
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def pack_bits(rows: list[list[int]], words: int) -> np.ndarray:
    m = np.zeros((len(rows), words), np.uint32)
    for i, r in enumerate(rows):
        for j in r:
            m[i, j // 32] |= np.uint32(1 << (j % 32))
    return m.view(np.int32)


def accept(parents, tokens, targets, root, keep):
    """(kept path, next token) of one tree; root None: a node without a parent needs no agreement."""
    paths = ancestors(parents)
    best: list[int] = []
    for path in paths:
        ok = all((root is None or tokens[i] == root) if parents[i] < 0 else tokens[i] == targets[parents[i]] for i in path)
        if ok and len(path) > len(best):
            best = path
    best = best[:keep]
    return best, (targets[best[-1]] if best else (-1 if root is None else root))


def tables_step(tables, held, lengths, grow, ring, head, tail, page):
    """One step of the page bookkeeping, request by request: (tables, ring, slots per request, head, tail)."""
    tables, ring = [list(r) for r in tables], list(ring)
    pool = len(ring)
    taken, given, slots = [], [], []
    for r, (h, t, g) in enumerate(zip(held, lengths, grow)):
        had, want = -(-h // page), -(-(t + g) // page)
        for k in range(had, want):
            tables[r][k] = ring[(head + len(taken)) % pool]
            taken.append(r)
        for k in range(want, had):
            given.append(tables[r][k])
        slots.append([tables[r][p // page] * page + p % page for p in range(t, t + g)])
    for i, x in enumerate(given):
        ring[(tail + i) % pool] = x
    return tables, ring, slots, head + len(taken), tail + len(given)


def attention(q, k, v, k_cache, v_cache, tables, lengths, starts, bits, scale=None):
    """(out, lse, allowed error of out, of lse) in 64 bits, request by request.

    bits: per request a bool [n, n] array of what a node sees, or None for a chain. The error that fp32 scores and
    sums with probabilities rounded to the inputs' type allow, with u = eps / 2 of that type:
      |out - ref| <= (u + 2 d) A + u |ref| + f,   A = sum_j w_j |v_j|  (w: exact weights)
    where u A is the rounding of the probabilities, u |ref| that of the result, and d bounds how far a score is off:
    dim products summed in fp32, in any order, are off by at most dim * 2^-24 * S with S = scale * sum |q||k|, the scaling, the
    shift by the maximum and exp2 by 2^-24 * 4 (|s| + |max| + 1) more; a weight then moves by at most exp(2 d) - 1, about 2 d,
    and the sum of the weights' rounding in fp32 adds 2^-24 per term, at most keys * 2^-24 relative. fp16 probabilities below
    2^-14 are off by up to 2^-25 instead (of a largest one of at least 2^7): f = 2^-32 sum_j |v_j| / l.
    A result below 2^-14 in fp16 is rounded by up to half a subnormal step, 2^-25, instead of u |ref|: f has that as well.
    (By arithmetic: of an exact -5.9195e-6, between 99 and 100 steps of 2^-24, the nearest number is 99 steps, -5.9009e-6; the
    right rounding is off by 1.87e-8, u |ref| is 0.29e-8, 2^-25 is 2.98e-8.)
    The log of the sum is off by 2 d, the sum's rounding (keys * 2^-24) and 2^-22 (|lse| + 1) of the logarithm and the shift.
    """
    q64, k64, v64 = q.double(), k.double(), v.double()
    kc, vc = k_cache, v_cache
    total, heads, dim = q.shape
    kv = k.shape[1]
    page = kc.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(total, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((total, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b, t in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        if n == 0:
            continue
        pages = torch.tensor([tables[b][x] for x in range(-(-t // page))], dtype=torch.int64, device=q.device)
        see = torch.ones(n, t + n, dtype=torch.bool, device=q.device)
        see[:, t:] = torch.ones(n, n, dtype=torch.bool, device=q.device).tril() if bits is None or bits[b] is None else bits[b].to(q.device)
        for g in range(kv):
            kk = torch.cat([kc[pages][:, :, g].reshape(-1, dim)[:t].double(), k64[lo:hi, g]])
            vv = torch.cat([vc[pages][:, :, g].reshape(-1, dim)[:t].double(), v64[lo:hi, g]])
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                s = (q64[lo:hi, h] @ kk.T) * scale
                s = torch.where(see, s, torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
                top = s.amax(-1, keepdim=True)
                top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
                e = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
                l = e.sum(-1, keepdim=True)
                w = torch.where(l > 0, e / l, torch.zeros_like(e))
                # A hidden value has no influence, not even as 0 * NaN.
                used = see.any(0)
                vz = torch.where(used[:, None], vv, torch.zeros_like(vv))
                if not bool(torch.isfinite(vz).all()):
                    o = torch.stack([w[i][see[i]] @ vv[see[i]] for i in range(n)])
                    a = torch.stack([w[i][see[i]] @ vv[see[i]].abs() for i in range(n)])
                    f = torch.stack([vv[see[i]].abs().sum(0) for i in range(n)])
                else:
                    o, a, f = w @ vz, w @ vz.abs(), see.double() @ vz.abs()
                out[lo:hi, h] = o
                lse[lo:hi, h] = torch.where(l > 0, top + torch.log(l), torch.full_like(l, -math.inf))[:, 0]
                big = torch.where(see, (q64[lo:hi, h].abs() @ kk.abs().nan_to_num(0, 0, 0).T) * abs(scale), torch.zeros_like(s)).amax(-1, keepdim=True)
                d = 2.0 ** -24 * (dim * big + 4 * (2 * big + 1))
                sub = 2.0 ** -32 * f / l.clamp(min=1e-300) + 2.0 ** -25 if q.dtype == torch.float16 else 0.0
                tol[lo:hi, h] = (u + 2 * d + (t + n) * 2.0 ** -24) * a + u * o.abs() + sub
                lse_tol[lo:hi, h] = (2 * d + (t + n) * 2.0 ** -24)[:, 0] + 2.0 ** -22 * (lse[lo:hi, h].abs().nan_to_num(0, 0, 0) + 1)
    return out, lse, tol, lse_tol
