"""Operators of the 4-bit cache at the edges of what their inputs may be."""

from __future__ import annotations

from fractions import Fraction

import pytest
import torch

import cache_util as U

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------------------ rows in and out
def _codes(x):
    """The codes of rows [n, 1, dim] as exact fractions give them (64 bits lose a minimum far below them, too), for offset and scale as encode has them."""
    _, scales, offsets = U.encode(x)
    codes = []
    for row, s, o in zip(x[:, 0].tolist(), scales[:, 0].tolist(), offsets[:, 0].tolist()):
        codes.append([min(15, max(0, round((Fraction(y) - Fraction(o[d // 32])) / Fraction(s[d // 32])))) for d, y in enumerate(row)])
    return torch.tensor(codes, device=x.device)[:, None], scales, offsets


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_codes_of_ties_beside_a_tiny_minimum(dtype, dim):
    """Halves of a step whose difference to the minimum rounds to a half of a step in fp32: what was lost decides, the bytes show it."""
    from actfold_b200.speculative import Int4Cache, write_cache_int4

    groups = []
    tinies = [2.0 ** -24, 3 * 2.0 ** -24] if dtype is HF else [2.0 ** -30, 2.0 ** -40, 5 * 2.0 ** -100, 2.0 ** -22]
    for step in (2.0, 6.0, 26.0, 1024.0):
        for tiny in tinies:
            for low in (tiny, -tiny, 0.0):
                x = step * torch.arange(32, dtype=torch.float64) / 2          # whole and half steps, 0 to 15.5
                x[0], x[31] = low, 15 * step
                groups += [x, (x - 15 * step) * (1 if low else -1)]           # (the second: a large minimum)
    x = torch.stack(groups).to(dtype).cuda()
    per = dim // 32
    n = -(-x.shape[0] // per)
    k = torch.cat([x, x[: n * per - x.shape[0]]]).view(n, 1, dim)
    v = k.flip(0).contiguous()
    cache = Int4Cache.empty(-(-n // 8), 8, 1, dim, dtype)
    cache.data.zero_()
    write_cache_int4(k, v, cache, torch.arange(n, device="cuda"))
    want = torch.zeros_like(cache.data)
    for part, rows in enumerate((k, v)):
        codes, scales, offsets = _codes(rows)
        for i in range(n):
            U.put(want, i, part, codes[i], scales[i], offsets[i])
    assert torch.equal(cache.data, want), (cache.data != want).nonzero()[:8]
