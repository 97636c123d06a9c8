"""Operators of the 4-bit cache at the edges of what their inputs may be."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

import cache_util as U
from test_cache_kernels_gpu import KINDS, _attention_case, _check_attention, _evict_case, _i32, _i64

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


# ------------------------------------------------------------------------------------------------ chains behind a window
def _seen_in_chain(n, t, bits, window, sinks):
    """[n, t + n]: a chain goes on where the cache ends, so the token at place t + i sees its last `window` places and the first `sinks`."""
    if bits is not None:
        return PREFIX_ONLY(n, t, bits, window, sinks)
    place, at = torch.arange(t + n)[None], t + torch.arange(n)[:, None]
    return (place <= at) & ((place > at - window) | (place < sinks) if window else True)


PREFIX_ONLY = U.visible


@pytest.mark.parametrize("window,sinks", [(4, 2), (1, 1), (16, 40), (33, 5), (20, 300)])
@pytest.mark.parametrize("dim,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("kind", KINDS)
def test_first_tokens_of_a_chain_stay_visible(monkeypatch, kind, dim, dtype, window, sinks):
    """An empty prefix, one shorter than the first tokens, one longer: all of the request's first tokens stay, wherever they lie."""
    monkeypatch.setattr(U, "visible", _seen_in_chain)
    for ls in ([0, 3, 130], [1, 0, 0], [35, 260, 2]):
        a, starts, bits = _attention_case(ls=ls, dim=dim, page=16, dtype=dtype, tree=False, seed=window + sinks, **KINDS[kind])
        _check_attention(a, ls, starts, bits, window, sinks)


@pytest.mark.parametrize("kind", KINDS)
def test_first_tokens_of_a_long_chain(monkeypatch, kind):
    """Rows far behind the first tokens, and values that are not finite among those and among tokens that only some windows hold."""
    monkeypatch.setattr(U, "visible", _seen_in_chain)
    shape = dict(KINDS[kind], ns=[{"8": 4, "16": 8, "128": 64, "256": 200}[kind]] * 8 + [300])
    ls = [0, 1, 5, 64, 300, 0, 0, 2, 0]
    a, starts, bits = _attention_case(ls=ls, dim=128, page=8, dtype=BF, tree=False, seed=9, **shape)
    _check_attention(a, ls, starts, bits, 70, 6)
    for node, x in ((2, math.inf), (100, math.nan), (150, -math.inf)):
        a["v"][starts[-2] + node, 1, 17 + node % 3] = x
    a["k"][starts[-2] + 4, 1, 3] = math.nan
    out = _check_attention(a, ls, starts, bits, 70, 3)
    assert out[starts[-2]:].isnan().any() and torch.isfinite(out[:, : shape["heads"] // 2]).all()


def test_a_prompt_may_be_cut_anywhere():
    """A chain in one call gives what it gives in pieces, each behind the rows that the cache holds of the pieces before."""
    from actfold_b200.speculative import Int4Cache, read_cache_int4, tree_attention_int4, write_cache_int4

    n, heads, kv, dim, window, sinks = 60, 4, 2, 64, 9, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    cache = Int4Cache.empty(9, 8, kv, dim, BF)
    slots = torch.arange(n, device="cuda")
    write_cache_int4(rand(n, kv, dim), rand(n, kv, dim), cache, slots)
    k, v = read_cache_int4(cache, slots)  # rows that 4 bits hold exactly: the same keys, cached or not
    q, tables = rand(n, heads, dim), _i32([list(range(9))])
    at = 0
    whole = tree_attention_int4(q, k, v, cache, tables, _i32([0]), _i32([0, n]), window=window, sinks=sinks)
    see = _seen_in_chain(n, 0, None, window, sinks).cuda()
    for h in range(heads):
        s = torch.where(see, q[:, h].double() @ k[:, h // 2].double().T * dim ** -0.5, -math.inf)
        w = torch.softmax(s, 1)
        # Probabilities and results rounded to 8 bits: half a step each, and a hair for fp32 (see U.attention).
        tol = 2.0 ** -8 * (w @ v[:, h // 2].double().abs()) * 1.01 + 2.0 ** -8 * (w @ v[:, h // 2].double()).abs()
        assert bool(((whole[:, h].double() - w @ v[:, h // 2].double()).abs() <= tol).all())
    for end in (3, 4, 11, 40, n):
        part = tree_attention_int4(q[at:end], k[at:end], v[at:end], cache, tables, _i32([at]), _i32([0, end - at]), window=window, sinks=sinks)
        # Both lie within 2^-7 of the largest value, by the same bound.
        assert bool(((part.double() - whole[at:end].double()).abs() <= 2.0 ** -6 * v.double().abs().max()).all())
        at = end


def test_attention_with_a_scale_below_fp32():
    """A scale that is no fp32 number but 0 is 0, not NaN where something is hidden."""
    from actfold_b200.speculative import tree_attention_int4

    for kind in KINDS:
        a, starts, bits = _attention_case(ls=[70, 300, 33], dim=64, page=16, dtype=BF, tree=True, seed=4, **KINDS[kind])
        zero = tree_attention_int4(**a, scale=0.0)
        for scale in (1e-50, -1e-50):
            assert torch.equal(tree_attention_int4(**a, scale=scale), zero)


# ------------------------------------------------------------------------------------------------ weights
def _given(q, keys, lse, window, sinks):
    """Sums over rows and heads of the group, of one request, in 64 bits; rows whose lse is -inf give nothing."""
    n, heads, dim = q.shape
    t, kv = keys.shape[:2]
    out = torch.zeros(kv, t, dtype=torch.float64, device=q.device)
    see = U.visible(n, t, None, window, sinks)[:, :t].to(q.device)
    for h in range(heads):
        x = (q[:, h, None].double() * keys[None, :, h * kv // heads].double()).sum(-1) * dim ** -0.5 - lse[:, h, None].double()
        out[h * kv // heads] += torch.where(see & (lse[:, h, None] != -math.inf), torch.exp(x), 0.0).sum(0)
    return out


@pytest.mark.parametrize("window,sinks", [(None, 0), (30, 2)])
@pytest.mark.parametrize("n,heads,kv", [(1, 7, 1), (1, 8, 1), (3, 4, 2), (13, 10, 2), (16, 8, 2)])
@pytest.mark.parametrize("dim,dtype", [(64, HF), (128, BF)])
def test_weights_of_keys_that_are_infinite(dim, dtype, n, heads, kv, window, sinks):
    """An infinite key gives what its scores say (0, an infinity or NaN), however many rows there are; rows without weight give nothing to any."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import Int4Cache, attention_weights, read_cache_int4, write_cache_int4

    t, page = 75, 16
    g = torch.Generator(device="cuda").manual_seed(n * heads)
    q = torch.randn(n, heads, dim, device="cuda", generator=g).abs().to(dtype)  # all positive: an infinite key's score is its infinity
    cache = Int4Cache.empty(6, page, kv, dim, dtype)
    keys = torch.randn(96, kv, dim, device="cuda", generator=g).to(dtype)
    write_cache_int4(keys, keys, cache, torch.arange(96, device="cuda"))
    keys = read_cache_int4(cache, torch.arange(96, device="cuda"))[0]
    nan = keys[:1].clone()
    nan[0, 0, 5] = math.nan
    write_cache_int4(nan, nan, cache, _i64([50]))
    held = read_cache_int4(cache, torch.arange(96, device="cuda"))[0]
    keys[1, 0, 3] = -math.inf
    keys[20, 0, 9] = math.inf
    keys[50, 0, 5] = math.nan
    keys[60, kv - 1, 0] = -math.inf
    keys[74, 0, 1], keys[74, 0, 2] = math.inf, -math.inf
    lse = torch.full((n, heads), 3.0, device="cuda") + torch.rand(n, heads, device="cuda", generator=g)
    st = DeviceStatus()
    for none in (False, True):
        if none:  # every other row, then all rows of a group
            lse[::2] = -math.inf
            lse[:, : heads // kv] = -math.inf
        for c, k in ((keys.view(6, page, kv, dim), keys), (cache, held)):
            w = attention_weights(q, c, _i32([list(range(6))]), _i32([t]), _i32([0, n]), lse, torch.zeros(1, kv, t, device="cuda"), window=window,
                                  sinks=sinks, status=st)
            st.check_status()
            want = _given(q, k[:t], lse, window or 0, sinks)
            # dim products in fp32 and an exponential of up to 2^6: 2^-23 (dim + 2^4) 2^6 relative, times e for the shift.
            near = (w[0].double() - want).abs() <= 2.0 ** -12 * want.abs()
            assert bool((near | (w[0] == want) | (w[0].isnan() & want.isnan())).all()), (w[0], want)
            if none:
                assert not w[0, 0].any()


def test_weights_report_lengths_without_pages():
    """Lengths that no page and no table can hold are reported, and nothing is added."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import Int4Cache, attention_weights

    q, lse = torch.ones(3, 4, 64, dtype=BF, device="cuda"), torch.zeros(3, 4, device="cuda")
    none, cache = Int4Cache.empty(0, 8, 2, 64, BF), Int4Cache.empty(2, 8, 2, 64, BF)
    rows = torch.zeros(0, 8, 2, 64, dtype=BF, device="cuda")
    for c, tables in ((none, _i32([[0, 0]])), (rows, _i32([[0, 0]])), (cache, torch.zeros(1, 0, dtype=torch.int32, device="cuda"))):
        for length in (0, 5, -1):
            st, w = DeviceStatus(), torch.ones(1, 2, 8, device="cuda")
            attention_weights(q, c, tables, _i32([length]), _i32([0, 3]), lse, w, status=st)
            assert int(st.status) == (4 if length else 0) and bool((w == 1).all())


def test_weights_end_when_a_wait_runs_out():
    """No attempts: every copy of keys counts as one that did not come. The call ends and says so, with copies in flight, and the next one is right."""
    from actfold_b200 import _lib
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import attention_weights, read_cache_int4

    ls = [9000, 9000, 3000, 1]
    a, starts, _ = _attention_case([4, 1, 30, 2], ls, 8, 2, 128, 16, BF, False, 5)  # (120 rows a head: more than are held at once)
    lse = torch.full((starts[-1], 8), 9.0, device="cuda")
    rows = read_cache_int4(a["cache"], torch.arange(a["cache"].pages * 16, device="cuda"))[0].view(-1, 16, 2, 128)
    st = DeviceStatus()

    def call(cache):
        return attention_weights(a["q"], cache, a["tables"], a["lengths"], a["starts"], lse, torch.zeros(4, 2, 9000, device="cuda"), status=st)

    good, good16 = call(a["cache"]), call(rows)
    st.check_status()
    _lib.check(_lib.load().af_tree_attention_wait_limit(0))
    try:
        for _ in range(20):
            call(a["cache"])
            with pytest.raises(TimeoutError):
                st.check_status()
        assert torch.equal(call(rows), good16)  # (rows of 16 bits come without a wait)
        st.check_status()
    finally:
        _lib.check(_lib.load().af_tree_attention_wait_limit(-1))
    assert torch.equal(call(a["cache"]), good)
    st.check_status()


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("held", [4, 16])
def test_evict_keeps_the_weights_of_requests_with_bad_lengths(held):
    """As their rows and their lengths, so that a caller who takes the result's weights over loses nothing."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import evict_cache

    for length in (-1, 10 ** 6, 34):  # negative, past the table, past the weights
        cache, _, tables, w = _evict_case(2, [32, 30], 2, 64, 8, BF, held, 2, extra=1)
        st = DeviceStatus()
        r = evict_cache(cache, tables, _i32([length, 30]), w, 20, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
        assert torch.equal(r.weights[:, 0], w[:, 0]) and r.lengths.tolist() == [length, 20]
        assert bool((r.kept[:, 0] == -1).all()) and not r.weights[:, 1, :, 20:].any()
