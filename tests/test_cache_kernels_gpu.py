"""Operators of the 4-bit cache against plain 64-bit forms. What is held in 4 bits, places and moved rows must be equal."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import cache_util as U

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _bits(x):
    return x.contiguous().view(torch.int16 if x.dtype in (BF, HF) else torch.int32) if x.is_floating_point() else x


def _same(a, b):
    """Equal values (0 and -0 alike), NaN in the same places."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("layers,n,heads,dim,page,dtype", [(None, 1, 1, 64, 8, BF), (None, 37, 4, 128, 16, BF), (3, 20, 5, 64, 48, HF), (2, 9, 32, 128, 64, HF),
                                                           (None, 130, 3, 64, 8, HF), (28, 6, 1, 128, 128, BF)])
def test_write_and_read(layers, n, heads, dim, page, dtype):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import Int4Cache, read_cache_int4, write_cache_int4

    g = torch.Generator(device="cuda").manual_seed(n + heads)
    pages = -(-n // page) + 2
    cache = Int4Cache.empty(pages, page, heads, dim, dtype, layers)
    cache.data.random_(0, 256, generator=g)
    before = cache.data.clone()
    lead = () if layers is None else (layers,)
    k, v = ((torch.randn(*lead, n, heads, dim, device="cuda", generator=g) * torch.exp(2 * torch.randn(n, heads, 1, device="cuda", generator=g))).to(dtype)
            for _ in range(2))
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n]
    slots[n // 3] = -1
    st = DeviceStatus()
    write_cache_int4(k, v, cache, slots, status=st)
    got = read_cache_int4(cache, slots, status=st)
    st.check_status()
    live = [i for i in range(n) if i != n // 3]
    for x, y in zip((k, v), got):
        want = U.values(*U.encode(x))
        assert _same(y[..., live, :, :], want[..., live, :, :]) and not y[..., n // 3, :, :].any()
    # The bytes are those of the layout, and no others are touched.
    want = before if layers is not None else before[None]
    for l in range(layers or 1):
        for part, x in enumerate((k, v)):
            codes, scales, offsets = U.encode(x[l] if layers is not None else x)
            for i in live:
                U.put(want[l], int(slots[i]), part, codes[i], scales[i], offsets[i])
    assert torch.equal(cache.data, want if layers is not None else want[0])
    assert _same(U.decoded(want[0], dtype)[0][slots[live]], got[0][..., live, :, :] if layers is None else got[0][0, live])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_groups_of_every_kind(dtype):
    """Equal values, zeros, halves of a step (ties), the type's extremes, subnormal numbers, infinities and NaN."""
    from actfold_b200.speculative import Int4Cache, read_cache_int4, write_cache_int4

    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    sub = 2.0 ** -24 if dtype is HF else 2.0 ** -133
    i = torch.arange(32, dtype=torch.float64)
    rows = [torch.zeros(32), torch.full((32,), 3.25), -i, i / 2, i * 15 / 31, torch.where(i == 0, top, -top), torch.where(i == 5, top, 0.0),
            torch.where(i < 16, -top, -top / 2), i * tiny, i * sub, i * sub * 4, torch.where(i == 31, math.inf, i), torch.where(i == 0, -math.inf, i),
            torch.where(i == 9, math.nan, i), torch.full((32,), math.inf), torch.where(i % 2 == 0, -0.0, 0.0), 7.5 * (i % 3), i % 31 - 7.5,
            torch.where(i == 0, -15.0, torch.where(i == 1, 2.0 ** -20, -(i % 16))), torch.where(i == 0, -7.5, torch.where(i == 1, 7.5, 2.0 ** -24)),
            torch.where(i == 3, 15.0, 0.5 + i % 15), 1000 + i]
    x = torch.stack([r.to(torch.float64) for r in rows]).to(dtype).cuda()
    n = x.shape[0]
    k = x.repeat(1, 2).view(n, 1, 64).contiguous()
    k[:, 0, 32:] = k[:, 0, 32:].flip(-1)
    v = k.flip(0).contiguous()
    cache = Int4Cache.empty(3, 8, 1, 64, dtype)
    slots = torch.arange(n, device="cuda")
    write_cache_int4(k, v, cache, slots)
    for a, b in zip(read_cache_int4(cache, slots), (k, v)):
        want = U.values(*U.encode(b))
        assert _same(a, want), (a != want).nonzero()
    got = read_cache_int4(cache, slots)[0][:, 0, :32]
    # (Row 5's range, twice the largest number, is past fp32's where the type is bf16.)
    assert got.isnan().all(1).nonzero()[:, 0].tolist() == ([5] if dtype is BF else []) + [11, 12, 13, 14] and not got.isinf().any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_error_is_half_a_step(dtype):
    """Off by at most half a step, and the roundings: of the scale by u of 15 steps, of the value by u of itself."""
    from actfold_b200.speculative import Int4Cache, read_cache_int4, write_cache_int4

    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(4000, 2, 128, device="cuda", generator=g).to(dtype)
    cache = Int4Cache.empty(250, 16, 2, 128, dtype)
    slots = torch.randperm(4000, device="cuda", generator=g)
    write_cache_int4(k, k, cache, slots)
    u = torch.finfo(dtype).eps / 2
    x = k.double().unflatten(-1, (4, 32))
    step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
    for y in read_cache_int4(cache, slots):
        y = y.double().unflatten(-1, (4, 32))
        assert bool(((y - x).abs() <= step * (1 + u) / 2 + 15 * u * step + u * y.abs()).all())


def test_rows_by_number_strides_and_bad_slots():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import Int4Cache, read_cache_int4, write_cache_int4

    g = torch.Generator(device="cuda").manual_seed(4)
    full = torch.randn(2, 40, 2, 5, 130, device="cuda", generator=g).to(HF)
    odd = full[:, :, 0, :, 1:129]                                   # rows that are not 16-byte aligned
    even = full.new_empty(2, 5, 40, 136).normal_(generator=g)[..., :128].transpose(1, 2)  # heads outside the rows
    big = torch.zeros(2, 6, 7, 2, 1280, dtype=torch.uint8, device="cuda")
    cache = Int4Cache(big[:, 1:5, 1:6], HF)                         # a part of a larger pool
    slots = _i64([[3, -1, 17], [63, 9, 30]])
    rows = _i32([[39, 0, -1], [0, 7, 7]])
    st = DeviceStatus()
    write_cache_int4(odd, even, cache, slots, rows=rows, status=st)
    st.check_status()
    k, v = read_cache_int4(cache, slots)
    assert k.shape == (2, 2, 3, 5, 128)
    for a, b in ((k, odd), (v, even)):
        want = U.values(*U.encode(b[:, rows.clamp(min=0).long()]))
        want[:, 0, 1:] = 0                                          # a negative slot; a negative row: the zeros that were there
        assert _same(a, want)
    assert not big[:, 0].any() and not big[:, 5].any() and not big[:, :, 0].any() and not big[:, :, 6].any()
    for call in (lambda: write_cache_int4(odd, even, cache, _i64([64]), rows=_i32([0]), status=st),
                 lambda: write_cache_int4(odd, even, cache, _i64([5]), rows=_i32([40]), status=st), lambda: read_cache_int4(cache, _i64([2 ** 40]), status=st)):
        call()
        with pytest.raises(RuntimeError):
            st.check_status()
    write_cache_int4(odd[:, :0], even[:, :0], cache, slots[:0, 0], status=st)
    assert read_cache_int4(cache, slots[:0])[0].shape == (2, 0, 3, 5, 128)
    st.check_status()


# ------------------------------------------------------------------------------------------------ eviction
def _evict_case(layers, ls, heads, dim, page, dtype, held, seed, extra=3):
    from actfold_b200.speculative import Int4Cache

    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-t // page) for t in ls]
    pool = sum(used) + 2
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((len(ls), max(1, *used) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, u in enumerate(used):
        tables[r, :u] = order[at:at + u]
        at += u
    lead = () if layers is None else (layers,)
    if held == 4:
        cache = Int4Cache.empty(pool, page, heads, dim, dtype, layers)
        cache.data.random_(0, 256, generator=g)
        rows = cache.data
        # One row of bytes per token and head: [.., pool * page, heads, 2, codes and pairs].
    else:
        cache = tuple(torch.randn(*lead, pool, page, heads, dim, device="cuda", generator=g).to(dtype) for _ in range(2))
        rows = cache
    w = torch.rand(*lead, len(ls), heads, max(1, *ls) + extra, device="cuda", generator=g)
    w = torch.where(w < 0.1, torch.zeros_like(w), (w * 50).round() / 50)  # many equal ones
    return cache, rows, tables, w


def _flat(cache, held, dtype):
    """[2 (keys, values), layers, slots, heads, dim]: what the cache holds, as whole numbers where they are codes."""
    if held == 16:
        return torch.stack([c if c.dim() == 5 else c[None] for c in cache]).flatten(2, 3)
    data = cache.data if cache.layers is not None else cache.data[None]
    out = []
    for d in data:
        pages, heads, blocks, size = d.shape
        dim = size // 10
        parts = d.reshape(pages, heads, blocks, 2, 5 * dim)
        codes = parts[..., : 4 * dim].reshape(pages, heads, blocks, 2, 8, dim // 2).clone()
        if dim == 128:
            codes[..., [2, 3, 6, 7], :] = codes[..., [2, 3, 6, 7], :].roll(32, -1)
        pairs = parts[..., 4 * dim:].reshape(pages, heads, blocks, 2, 8, dim // 8)
        out.append(torch.cat([codes, pairs], -1).permute(3, 0, 2, 4, 1, 5).reshape(2, -1, heads, dim // 2 + dim // 8))
    return torch.stack(out, 1)


@pytest.mark.parametrize("layers,ls,heads,dim,page,dtype,held,keep,sinks,recent", [
    (None, [40], 1, 64, 8, BF, 16, 20, 4, 5), (None, [40], 1, 64, 8, BF, 4, 20, 4, 5), (3, [100, 7, 0, 64, 65], 2, 128, 16, HF, 4, 64, 3, 10),
    (3, [100, 7, 0, 64, 65], 2, 128, 16, HF, 16, 64, 3, 10), (2, [5000, 3001], 1, 64, 48, BF, 4, 2999, 0, 0), (1, [9000], 2, 128, 64, BF, 4, 1, 0, 1),
    (1, [9000], 1, 128, 64, BF, 16, 8999, 1, 700), (28, [300, 280], 4, 128, 128, HF, 4, 150, 4, 30), (28, [1500] * 3, 4, 128, 16, BF, 16, 777, 2, 32),
    (None, [33, 12], 3, 64, 8, HF, 4, 0, 0, 0), (None, [20, 21], 2, 128, 8, BF, 4, 20, 12, 8), (40, [260, 500], 4, 64, 16, HF, 4, 200, 4, 8),
    (None, [3000], 1, 40, 24, torch.float32, 16, 1024, 4, 256)])
def test_evict(layers, ls, heads, dim, page, dtype, held, keep, sinks, recent):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import evict_cache

    cache, _, tables, w = _evict_case(layers, ls, heads, dim, page, dtype, held, keep + len(ls))
    before = _flat(cache, held, dtype)
    st = DeviceStatus()
    r = evict_cache(cache, tables, _i32(ls), w, keep, sinks=sinks, recent=recent, status=st)
    st.check_status()
    after = _flat(cache, held, dtype)
    assert r.lengths.tolist() == [min(t, keep) for t in ls]
    assert r.kept.shape == (*w.shape[:-1], keep) and r.weights.shape == w.shape
    kept, given, old = (x if layers is not None else x[None] for x in (r.kept, r.weights, w))
    want = before.clone()
    for l in range(layers or 1):
        for b, t in enumerate(ls):
            place = torch.arange(max(t, 1), device="cuda")
            slot = tables[b].long()[place // page] * page + place % page
            for h in range(heads):
                places = U.evict(old[l, b, h, :t].tolist(), keep, sinks, recent)
                assert kept[l, b, h].tolist() == places + [-1] * (keep - len(places))
                assert torch.equal(given[l, b, h, :len(places)], old[l, b, h, places]) and not given[l, b, h, len(places):].any()
                if t > keep:
                    want[:, l, slot[:keep], h] = before[:, l, slot[places], h]
    assert torch.equal(_bits(after), _bits(want))


def test_evict_weights_of_every_kind():
    """Negative weights, zeros of both signs, infinities and NaN; a weight that all tokens share."""
    from actfold_b200.speculative import evict_cache

    for w in ([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, 0.0, -0.0, 2.0, math.nan, 1e-45], [1.5] * 12, [-0.0, 0.0] * 6):
        cache, _, tables, _ = _evict_case(None, [12], 1, 64, 8, BF, 4, 1)
        for keep in range(12):
            r = evict_cache(cache, tables, _i32([12]), torch.tensor(w, device="cuda").view(1, 1, 12), keep, sinks=min(1, keep))
            assert r.kept[0, 0].tolist() == U.evict(w, keep, min(1, keep), 0), (w, keep)


def test_evict_reports_bad_lengths_and_pages():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import evict_cache

    st = DeviceStatus()
    for ls in ([-1, 30], [10 ** 6, 30], [34, 30]):  # negative, past the table, past the weights
        cache, _, tables, w = _evict_case(None, [32, 30], 2, 64, 8, BF, 4, 2, extra=1)
        before = cache.data.clone()
        r = evict_cache(cache, tables, _i32(ls), w, 20, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
        assert r.lengths.tolist() == [ls[0], 20] and (r.kept[0] == -1).all() and (r.kept[1] >= 0).all()
        mine = tables[0, :4].long()
        assert torch.equal(cache.data[mine], before[mine])
    for page in (-1, 10 ** 6):
        cache, _, tables, w = _evict_case(None, [32, 30], 2, 64, 8, BF, 4, 2)
        tables[0, 3] = page
        r = evict_cache(cache, tables, _i32([32, 30]), w, 20, status=st)
        assert r.lengths.tolist() == [20, 20]
        with pytest.raises(RuntimeError):
            st.check_status()


# ------------------------------------------------------------------------------------------------ attention
def _attention_case(ns, ls, heads, kv, dim, page, dtype, tree, seed, extra_rows=0):
    """Keys with a few strong channels; scattered pages; random bytes in the places behind a request's last token."""
    import tree_util as T
    from actfold_b200.speculative import Int4Cache, write_cache_int4

    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-t // page) for t in ls]
    pool = sum(used) + 2
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((len(ls), max(1, *used) + 1), -1, dtype=torch.int32, device="cuda")
    slots, at = [], 0
    for r, (u, t) in enumerate(zip(used, ls)):
        tables[r, :u] = order[at:at + u]
        at += u
        place = torch.arange(t, device="cuda")
        slots.append(tables[r].long()[place // page] * page + place % page)
    slots = torch.cat(slots)
    cache = Int4Cache.empty(pool, page, kv, dim, dtype)
    cache.data.random_(0, 256, generator=g)
    strong = torch.where(torch.rand(kv, dim, device="cuda", generator=g) < 0.05, 3.0, 1.0)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    write_cache_int4((rand(slots.numel(), kv, dim) * strong).to(dtype), rand(slots.numel(), kv, dim).to(dtype), cache, slots)
    total = sum(ns) + extra_rows
    starts = [0, *np.cumsum(ns).tolist()]
    bits = mask = None
    if tree:
        paths = [T.ancestors(T.random_parents(n, rng)) for n in ns]
        words = max(1, -(-max(ns) // 32))
        mask = torch.zeros(total, words, dtype=torch.int32, device="cuda")
        bits = []
        for b, p in enumerate(paths):
            m = torch.zeros(ns[b], ns[b], dtype=torch.bool)
            for i, row in enumerate(p):
                m[i, row] = True
            bits.append(m)
            if ns[b]:
                mask[starts[b]:starts[b + 1]] = torch.from_numpy(T.pack_bits(p, words)).cuda()
    a = dict(q=rand(total, heads, dim).to(dtype), k=(rand(total, kv, dim) * strong).to(dtype), v=rand(total, kv, dim).to(dtype), cache=cache,
             tables=tables, lengths=_i32(ls), starts=_i32(starts), mask=mask)
    return a, starts, bits


def _check_attention(a, ls, starts, bits, window=None, sinks=0, **kw):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention_int4

    st = DeviceStatus()
    total, heads = a["q"].shape[:2]
    lse = torch.full((total, heads), 7.0, device="cuda")
    out = tree_attention_int4(**a, window=window, sinks=sinks, lse=lse, status=st, **kw)
    st.check_status()
    n = starts[-1]
    want, want_lse, tol, lse_tol = U.attention(a["q"], a["k"], a["v"], a["cache"].data, a["cache"].dtype, a["tables"].tolist(), ls, starts, bits,
                                               window or 0, sinks, kw.get("scale"))
    assert U.close(out[:n], want[:n], tol[:n]), ((out[:n].double() - want[:n]).abs() / tol[:n]).nan_to_num(0).max()
    assert U.close(lse[:n], want_lse[:n], lse_tol[:n])
    assert bool((lse[n:] == 7.0).all())
    return out


@pytest.mark.parametrize("ns,ls,heads,kv,dim,page,dtype,tree", [
    ([1], [523], 28, 4, 128, 16, BF, False), ([1], [0], 4, 4, 64, 8, HF, False), ([1, 1, 1, 1], [1, 31, 32, 33], 8, 2, 128, 8, BF, False),
    ([1] * 9, [2000, 90, 0, 700, 64, 1, 1024, 1025, 300], 28, 4, 128, 64, BF, False), ([1] * 3, [6000, 5, 4000], 12, 1, 64, 48, HF, False),
    ([5, 0, 17, 1], [100, 50, 333, 2000], 32, 32, 128, 64, BF, True), ([64, 40], [900, 4100], 8, 8, 128, 64, BF, True),
    ([33, 70], [40, 1500], 28, 4, 128, 16, HF, True), ([3, 2], [500, 0], 16, 2, 64, 24, HF, False), ([100, 31, 0], [77, 0, 9], 5, 5, 128, 128, BF, False),
    ([1, 2], [300, 1200], 64, 1, 64, 16, BF, False), ([2], [3000], 80, 1, 128, 32, HF, True), ([8] * 40, list(range(0, 400, 10)), 4, 4, 64, 16, BF, True)])
def test_attention(ns, ls, heads, kv, dim, page, dtype, tree):
    a, starts, bits = _attention_case(ns, ls, heads, kv, dim, page, dtype, tree, sum(ns) + heads)
    _check_attention(a, ls, starts, bits)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 0), (16, 1), (32, 4), (100, 0), (100, 40), (128, 128), (1000, 8), (5000, 4)])
@pytest.mark.parametrize("ns,ls,heads,kv,dim,page,dtype,tree", [
    ([1] * 6, [0, 1, 40, 129, 2000, 1023], 8, 2, 128, 16, BF, False), ([6, 40, 1], [90, 300, 1500], 4, 4, 64, 8, HF, False),
    ([20, 64, 3], [0, 700, 1300], 14, 2, 128, 48, BF, True)])
def test_attention_window(ns, ls, heads, kv, dim, page, dtype, tree, window, sinks):
    a, starts, bits = _attention_case(ns, ls, heads, kv, dim, page, dtype, tree, sum(ns) + window)
    _check_attention(a, ls, starts, bits, window, sinks)


# ------------------------------------------------------------------------------------------------ weights
@pytest.mark.parametrize("ns,ls,heads,kv,dim,page,dtype,held,window,sinks", [
    ([1], [1500], 28, 4, 128, 16, BF, 4, None, 0), ([1, 0, 5, 12], [1, 40, 0, 700], 8, 2, 64, 8, HF, 4, None, 0),
    ([3] * 9, [2000, 90, 0, 700, 64, 1, 1024, 33, 31], 28, 4, 128, 64, BF, 4, None, 0), ([3] * 5, [2000, 90, 15, 16, 17], 32, 32, 128, 64, BF, 16, None, 0),
    ([9, 1, 2], [300, 1, 77], 12, 1, 64, 48, HF, 16, None, 0), ([4, 9, 1], [600, 100, 40], 10, 5, 128, 24, HF, 4, 50, 4),
    ([4, 9, 1], [600, 100, 40], 10, 5, 64, 24, BF, 16, 5, 0), ([40, 2], [3000, 5], 4, 4, 128, 16, BF, 4, 700, 100), ([200], [129], 14, 2, 128, 8, BF, 4, None, 0)])
def test_weights(ns, ls, heads, kv, dim, page, dtype, held, window, sinks):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import attention_weights, read_cache_int4

    a, starts, _ = _attention_case(ns, ls, heads, kv, dim, page, dtype, False, sum(ls) + heads, extra_rows=2)
    slots = [a["tables"][b].long()[torch.arange(t, device="cuda") // page] * page + torch.arange(t, device="cuda") % page for b, t in enumerate(ls)]
    pool = a["cache"].pages * page
    keys = read_cache_int4(a["cache"], torch.arange(pool, device="cuda"))[0]
    cache = a["cache"] if held == 4 else keys.view(-1, page, kv, dim)
    g = torch.Generator(device="cuda").manual_seed(9)
    lse = 5 + 2 * torch.randn(starts[-1] + 2, heads, device="cuda", generator=g)
    lse[0, 0] = -math.inf
    wide = torch.rand(len(ls), kv + 1, max(ls) + 40, device="cuda", generator=g)
    w = wide[:, :kv, 1: max(ls) + 4]
    before = wide.clone()
    st = DeviceStatus()
    got = attention_weights(a["q"], cache, a["tables"], a["lengths"], a["starts"], lse, w, window=window, sinks=sinks, status=st)
    st.check_status()
    assert got is w
    want, tol = U.weights(a["q"], keys, slots, ls, starts, lse, before[:, :kv, 1: max(ls) + 4], window or 0, sinks)
    assert U.close(w, want, tol), ((w.double() - want).abs() / tol).nan_to_num(0).max()
    wide[:, :kv, 1: max(ls) + 4] = before[:, :kv, 1: max(ls) + 4]
    assert torch.equal(wide, before)  # nothing beside
    for b, t in enumerate(ls):
        assert torch.equal(got[b, :, t:], before[b, :kv, 1 + t: max(ls) + 4])


def test_weights_are_those_of_the_attention():
    """Every row's weights over the prefix and its own nodes sum to one: what the prefix is given is what the chain's tree is not."""
    from actfold_b200.speculative import attention_weights, tree_attention_int4

    ls, heads, kv = [700, 64, 1], 8, 2
    a, starts, _ = _attention_case([1, 1, 1], ls, heads, kv, 128, 16, BF, False, 5)
    lse = torch.empty(3, heads, device="cuda")
    tree_attention_int4(**a, lse=lse)
    w = torch.zeros(3, kv, 700, device="cuda")
    attention_weights(a["q"], a["cache"], a["tables"], a["lengths"], a["starts"], lse, w)
    own = torch.einsum("bhd,bhd->bh", a["q"].double(), a["k"].double().repeat_interleave(heads // kv, 1)) * 128 ** -0.5
    left = (1 - torch.exp(own - lse.double())).view(3, kv, -1).sum(-1)
    assert bool(((w.double().sum(-1) - left).abs() <= 2.0 ** -14).all())  # 700 keys, scores below 32: 2^-23 * 128 * 32 * 4 terms


# Shapes that reach every kernel: 1 to 8 rows a head, 9 to 16, 17 to 128 (one row tile), more (two).
KINDS = {"8": dict(ns=[1, 3, 1], heads=4, kv=2), "16": dict(ns=[5, 9, 3], heads=4, kv=2), "128": dict(ns=[30, 40, 7], heads=4, kv=2),
         "256": dict(ns=[90, 20, 100], heads=4, kv=2)}


@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 3)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_values_that_are_not_finite(kind, tree, window, sinks, dim, dtype):
    """NaN and infinities in keys and values, cached and drafted, reach the rows that see them and no others."""
    from actfold_b200.speculative import write_cache_int4

    ls = [200, 65, 130]
    a, starts, bits = _attention_case(ls=ls, dim=dim, page=16, dtype=dtype, tree=tree, seed=len(kind) + dim, **KINDS[kind])
    kv = KINDS[kind]["kv"]
    g = torch.Generator(device="cuda").manual_seed(1)
    # Cached: a value of request 0 that only some windows hold, one among the sinks, a key of request 1.
    for r, place, part, d, x in ((0, 200 - 45, 1, 40, math.nan), (0, 1, 1, 3, math.inf), (1, 30, 0, 9, math.nan), (2, 129, 1, 20, -math.inf)):
        k, v = torch.randn(1, kv, dim, device="cuda", generator=g).to(dtype), torch.randn(1, kv, dim, device="cuda", generator=g).to(dtype)
        (k, v)[part][0, 1, d] = x
        write_cache_int4(k, v, a["cache"], a["tables"][r].long()[place // 16] * 16 + place % 16 + _i64([0]))
    # Drafted: values and a key of nodes that not all see.
    for r, node, part, d, x in ((0, -1, 1, 5, math.nan), (1, KINDS[kind]["ns"][1] // 2, 1, 50, math.inf), (1, KINDS[kind]["ns"][1] // 2 + 1, 1, 50, -math.inf),
                                (2, -1, 0, 7, math.nan)):
        lo, hi = starts[r], starts[r + 1]
        (a["k"], a["v"])[part][hi - 1 if node < 0 else lo + node, 1, d] = x
    out = _check_attention(a, ls, starts, bits, window, sinks)
    assert out.isnan().any() and torch.isfinite(out[:, : KINDS[kind]["heads"] // 2]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_strided_tensors(kind):
    """Rows, tables, lengths and results that are parts of larger tensors, and rows that are not 16-byte aligned."""
    ls = [70, 300, 33]
    for shift in (0, 1):
        a, starts, bits = _attention_case(ls=ls, dim=64, page=24, dtype=HF, tree=True, seed=3, extra_rows=2, **KINDS[kind])
        total, heads = a["q"].shape[:2]
        wide = torch.zeros(total, 3, heads + 2, 72, dtype=HF, device="cuda")
        q, k, v = (wide[:, i, : x.shape[1], shift:64 + shift].copy_(x) for i, x in enumerate((a["q"], a["k"], a["v"])))
        tables = torch.full((3, 2 * a["tables"].shape[1]), 10 ** 6, dtype=torch.int32, device="cuda")[:, ::2].copy_(a["tables"])
        lengths = torch.zeros(6, dtype=torch.int32, device="cuda")[::2].copy_(a["lengths"])
        mask = torch.full((total, 2 * a["mask"].shape[1]), -1, dtype=torch.int32, device="cuda")[:, : a["mask"].shape[1]].copy_(a["mask"])
        big = torch.full((total, heads, 2, 64), 5.0, dtype=HF, device="cuda")
        b = dict(a, q=q, k=k, v=v, tables=tables, lengths=lengths, mask=mask)
        out = _check_attention(b, ls, starts, bits, 50, 2, out=big[:, :, 1])
        assert out.data_ptr() == big[:, :, 1].data_ptr()
        assert bool((big[:, :, 0] == 5.0).all()) and bool((big[starts[-1]:] == 5.0).all())


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.5, 1e-4])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales(kind, scale):
    ls = [70, 300, 33]
    a, starts, bits = _attention_case(ls=ls, dim=128, page=16, dtype=HF if scale > 1 else BF, tree=True, seed=4, **KINDS[kind])
    _check_attention(a, ls, starts, bits, 100, 1, scale=scale)


def test_attention_with_rows_that_see_nothing():
    """Masks without a bit over an empty prefix, bits behind the tree's end, a mask of ones."""
    from actfold_b200.speculative import tree_attention_int4

    for kind in KINDS:
        a, starts, _ = _attention_case(ls=[0, 40, 5], dim=64, page=8, dtype=BF, tree=False, seed=5, **KINDS[kind])
        words = 4
        a["mask"] = torch.full((starts[-1], words), -1, dtype=torch.int32, device="cuda")  # ones, behind the end too
        n = KINDS[kind]["ns"]
        bits = [torch.ones(x, x, dtype=torch.bool) for x in n]
        _check_attention(a, [0, 40, 5], starts, bits)
        a["mask"][0] = 0
        bits[0][0] = False
        a["mask"][starts[1]] = 0
        bits[1][0] = False
        out = _check_attention(a, [0, 40, 5], starts, bits)
        assert not out[0].any()
        lse = torch.zeros(starts[-1], a["q"].shape[1], device="cuda")
        tree_attention_int4(**a, lse=lse)
        assert bool((lse[0] == -math.inf).all()) and torch.isfinite(lse[1:]).all()


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 2), (64, 0), (257, 5)])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_windows_with_any_bits(kind, window, sinks):
    """Nodes that see others but not themselves, or none: their windows reach to the last `window` tokens."""
    lengths = [window + 128, 384 + window, window + 31]  # the window's first token is the first, or last, of a unit
    a, starts, _ = _attention_case(ls=lengths, dim=128, page=16, dtype=BF, tree=False, seed=window, **KINDS[kind])
    n = KINDS[kind]["ns"]
    g = torch.Generator().manual_seed(window)
    bits = [torch.rand(x, x, generator=g) < torch.rand(x, 1, generator=g) for x in n]
    words = -(-max(n) // 32)
    a["mask"] = torch.zeros(starts[-1], words, dtype=torch.int32, device="cuda")
    for b, m in enumerate(bits):
        m[0] = False
        full = torch.zeros(n[b], 32 * words, dtype=torch.int64)
        full[:, :n[b]] = m
        packed = (full.view(n[b], words, 32) << torch.arange(32)).sum(2)
        a["mask"][starts[b]:starts[b + 1]] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).cuda()
    _check_attention(a, lengths, starts, bits, window, sinks)


def test_offsets_past_32_bits():
    """Pages, heads and layers that lie gigabytes apart give what a compact cache gives."""
    from actfold_b200.speculative import Int4Cache, attention_weights, evict_cache, read_cache_int4, tree_attention_int4, write_cache_int4

    layers, pages, page, kv, dim = 2, 3, 24, 2, 128
    blocks = page // 8
    far = torch.empty(5 << 31, dtype=torch.uint8, device="cuda")
    strides = ((1 << 32) + (1 << 31) + 16, (1 << 30) + 32, (1 << 29) + 48, 10 * dim, 1)
    assert sum((x - 1) * s for x, s in zip((layers, pages, kv, blocks, 10 * dim), strides)) < far.numel()
    caches = [Int4Cache(far.as_strided((layers, pages, kv, blocks, 10 * dim), strides), BF), Int4Cache.empty(pages, page, kv, dim, BF, layers=layers)]
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(layers, pages * page, kv, dim, device="cuda", generator=g).to(BF) for _ in range(2))
    slots = torch.randperm(pages * page, device="cuda", generator=g)
    tables, lengths = _i32([[2, 0, 1]]), _i32([70])
    results = []
    for cache in caches:
        write_cache_int4(k, v, cache, slots)
        got = [*read_cache_int4(cache, slots)]
        for n, heads in ((1, 4), (20, 8)):
            starts, q = _i32([0, n]), k[0, :n].repeat(1, heads // kv, 1)
            lse, w = torch.zeros(n, heads, device="cuda"), torch.zeros(layers, 1, kv, 72, device="cuda")
            for l in range(layers):
                got.append(tree_attention_int4(q, k[1, :n], v[1, :n], cache[l], tables, lengths, starts, lse=lse))
                attention_weights(q, cache[l], tables, lengths, starts, lse, w[l])
            got += [lse, w]
        got += [*evict_cache(cache, tables, lengths, w, 40, 1, 8), *read_cache_int4(cache, slots)]
        results.append(got)
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(*results))
    # The same of 16-bit keys.
    strides = ((1 << 31) + (1 << 30) + 8, (1 << 29) + 16, kv * dim, dim, 1)
    results = []
    for keys in (far.view(BF).as_strided((layers, pages, page, kv, dim), strides), torch.empty(layers, pages, page, kv, dim, dtype=BF, device="cuda")):
        keys.copy_(k.view(keys.shape))
        w = torch.zeros(layers, 1, kv, 72, device="cuda")
        for l in range(layers):
            attention_weights(q, keys[l], tables, lengths, starts, lse, w[l])
        results.append([w, *evict_cache((keys, v.view(keys.shape).clone()), tables, lengths, w, 40, 1, 8), keys])
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(*results))


@pytest.mark.parametrize("ns,ls,heads,kv,window", [([1], [30000], 7, 1, None), ([2] * 300, [90 + i for i in range(300)], 4, 2, None), ([1] * 50, [5000] * 50, 2, 2, 900),
                                                   ([20], [20000], 4, 1, None), ([60, 64], [9000, 7000], 8, 2, None), ([64] * 40, [300] * 40, 2, 2, 128)])
def test_attention_of_long_rows_and_many_requests(ns, ls, heads, kv, window):
    """Rows that many CTAs share, CTAs with many rows; the same bits in every run."""
    from actfold_b200.speculative import tree_attention_int4

    a, starts, bits = _attention_case(ns, ls, heads, kv, 128, 16, BF, False, 6)
    out = _check_attention(a, ls, starts, bits, window)
    for _ in range(3):
        assert torch.equal(_bits(tree_attention_int4(**a, window=window)), _bits(out))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_reports_bad_values(kind):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention_int4

    ls = [70, 300, 33]
    a, starts, bits = _attention_case(ls=ls, dim=64, page=16, dtype=BF, tree=False, seed=7, **KINDS[kind])
    good = tree_attention_int4(**a)
    st = DeviceStatus()
    for r, x in ((0, -1), (2, 10 ** 7)):  # lengths that are none: the request is left out
        lengths = a["lengths"].clone()
        lengths[r] = x
        out = torch.full_like(good, 3.0)
        tree_attention_int4(**{**a, "lengths": lengths}, out=out, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
        mine = torch.zeros(starts[-1], dtype=torch.bool, device="cuda")
        mine[starts[r]:starts[r + 1]] = True
        assert bool((out[mine] == 3.0).all()) and torch.allclose(out[~mine].float(), good[~mine].float(), rtol=2 ** -6, atol=2 ** -6)
    for bad in ([0, starts[2], starts[1], starts[3]], [0, starts[1], starts[2], starts[3] + 1], [-1, *starts[1:]]):
        tree_attention_int4(**{**a, "starts": _i32(bad)}, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
    for page in (-1, 10 ** 6):  # read as zeros
        tables = a["tables"].clone()
        tables[1, 3] = page
        out = tree_attention_int4(**{**a, "tables": tables}, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
        assert torch.equal(_bits(out[: starts[1]]), _bits(good[: starts[1]])) and torch.isfinite(out).all()


@pytest.mark.parametrize("kind", [*KINDS, "long"])
def test_attention_ends_when_a_wait_runs_out(kind):
    """No attempt but the first for every wait: the call ends and says so, or no wait was long (an attempt sleeps some microseconds); the
    next call is right. Values that are not finite in all of a long chain make row ends, and so some waits, long for certain."""
    from actfold_b200 import _lib
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention_int4

    ls = [3000, 900, 1400]
    shape = dict(ns=[1500, 3, 900], heads=4, kv=2) if kind == "long" else KINDS[kind]
    a, starts, bits = _attention_case(ls=ls, dim=128, page=16, dtype=BF, tree=False, seed=8, **shape)
    st = DeviceStatus()
    v = a["v"].clone()
    if kind == "long":
        v[::64] = math.inf
    _lib.check(_lib.load().af_tree_attention_wait_limit(0))
    try:
        out = tree_attention_int4(**{**a, "v": v}, status=st)
        ran_out = bool(int(st.status) & 1)
        if kind == "long":
            assert ran_out
        if ran_out:
            with pytest.raises(TimeoutError):
                st.check_status()
    finally:
        _lib.check(_lib.load().af_tree_attention_wait_limit(-1))
    if kind != "long":
        good = _check_attention(a, ls, starts, bits)
        assert ran_out or torch.equal(_bits(out), _bits(good))
    else:
        assert torch.isfinite(tree_attention_int4(**a, status=st)).all()
    st.check_status()


def test_weights_of_every_kind_of_row():
    """Keys that are not finite, rows without weight, more rows than are held at once; the same bits in every run."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import attention_weights, read_cache_int4, write_cache_int4

    ns, ls, heads, kv = [3, 40], [90, 200], 8, 2
    a, starts, _ = _attention_case(ns, ls, heads, kv, 64, 16, HF, False, 11)
    k = torch.zeros(1, kv, 64, dtype=HF, device="cuda")
    k[0, 1, 5] = math.nan
    write_cache_int4(k, k, a["cache"], a["tables"][0, 1].long() * 16 + _i64([3]))  # place 19 of request 0
    lse = torch.full((43, heads), 2.5, device="cuda")
    lse[1] = -math.inf
    lse[7] = math.inf
    runs = []
    for held in (4, 16):
        keys = read_cache_int4(a["cache"], torch.arange(a["cache"].pages * 16, device="cuda"))[0]
        cache = a["cache"] if held == 4 else keys.view(-1, 16, kv, 64)
        for window, sinks in ((None, 0), (30, 2)):
            slots = [a["tables"][b].long()[torch.arange(t, device="cuda") // 16] * 16 + torch.arange(t, device="cuda") % 16 for b, t in enumerate(ls)]
            want, tol = U.weights(a["q"], keys, slots, ls, starts, lse, torch.zeros(2, kv, 200, device="cuda"), window or 0, sinks)
            got = [attention_weights(a["q"], cache, a["tables"], a["lengths"], a["starts"], lse, torch.zeros(2, kv, 200, device="cuda"), window=window, sinks=sinks)
                   for _ in range(2)]
            assert torch.equal(got[0].nan_to_num(7.0), got[1].nan_to_num(7.0))
            if window is None:
                assert got[0][0, 1, 19].isnan() and torch.isfinite(got[0][0, 0]).all()
                want[0, 1, 19] = math.nan
            assert U.close(got[0], want, tol)
    st = DeviceStatus()
    w = torch.zeros(2, kv, 150, device="cuda")
    attention_weights(a["q"], a["cache"], a["tables"], a["lengths"], a["starts"], lse, w, status=st)  # 200 places do not fit into 150
    with pytest.raises(RuntimeError):
        st.check_status()
    assert not w[1].any() and w[0, 0, :90].all()
    for bad in ([0, 40, 3], [0, 3, 44]):
        attention_weights(a["q"], a["cache"], a["tables"], a["lengths"], _i32(bad), lse, torch.zeros(2, kv, 200, device="cuda"), status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
    for cache in (a["cache"], keys.view(-1, 16, kv, 64)):
        tables = a["tables"].clone()
        tables[1, 2] = 10 ** 6
        attention_weights(a["q"], cache, tables, a["lengths"], a["starts"], lse, torch.zeros(2, kv, 200, device="cuda"), status=st)
        with pytest.raises(RuntimeError):
            st.check_status()


# ------------------------------------------------------------------------------------------------ together
def test_steps_of_a_batch_over_its_budget():
    """Prompts in, then steps of one token: attention, weights, rows written, eviction, pages back. A plain loop keeps lists of rows."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import Int4Cache, attention_weights, block_tables, evict_cache, tree_attention_int4, write_cache_int4

    layers, kv, heads, dim, page, keep, sinks, recent, pool = 3, 2, 4, 64, 8, 24, 2, 6, 40
    prompts = [30, 9, 17, 24]
    n = len(prompts)
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    st = DeviceStatus()
    cache = Int4Cache.empty(pool, page, kv, dim, BF, layers)
    tables = torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    free, span = torch.arange(pool, dtype=torch.int32, device="cuda"), _i64([0, pool])
    weights = torch.zeros(layers, n, kv, 64, device="cuda")
    k, v = rand(layers, sum(prompts), kv, dim), rand(layers, sum(prompts), kv, dim)
    new = block_tables(tables, _i32([0] * n), _i32(prompts), free, span, page, sum(prompts), status=st)
    write_cache_int4(k, v, cache, new.slots, status=st)
    span, lengths = new.free_range, new.totals
    vk, vv = (U.values(*U.encode(x)) for x in (k, v))
    at = [0, *np.cumsum(prompts).tolist()]
    kept = [[[[(vk[l, i, h], vv[l, i, h]) for i in range(at[r], at[r + 1])] for h in range(kv)] for r in range(n)] for l in range(layers)]
    given = [[[[0.0] * p for _ in range(kv)] for p in prompts] for _ in range(layers)]
    for step in range(4):
        old = lengths
        q, k, v = rand(layers, n, heads, dim), rand(layers, n, kv, dim), rand(layers, n, kv, dim)
        starts = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        for l in range(layers):
            lse = torch.empty(n, heads, device="cuda")
            out = tree_attention_int4(q[l], k[l], v[l], cache[l], tables, lengths, starts, lse=lse, status=st)
            attention_weights(q[l], cache[l], tables, lengths, starts, lse, weights[l], status=st)
            for r in range(n):
                for h in range(heads):
                    gk = h * kv // heads
                    kk = torch.stack([x for x, _ in kept[l][r][gk]] + [k[l, r, gk]]).double()
                    ww = torch.stack([x for _, x in kept[l][r][gk]] + [v[l, r, gk]]).double()
                    p = torch.softmax(kk @ q[l, r, h].double() * dim ** -0.5, 0)
                    assert torch.allclose(out[r, h].double(), p @ ww, rtol=2 ** -7, atol=2 ** -6)
                    for i, x in enumerate(p[:-1].tolist()):
                        given[l][r][gk][i] += x
        grown = block_tables(tables, lengths, torch.ones_like(lengths), free, span, page, n, status=st)
        write_cache_int4(k, v, cache, grown.slots, status=st)
        vk, vv = (U.values(*U.encode(x)) for x in (k, v))
        for l in range(layers):
            for r in range(n):
                for h in range(kv):
                    kept[l][r][h].append((vk[l, r, h], vv[l, r, h]))
                    given[l][r][h].append(0.0)
        span = grown.free_range
        e = evict_cache(cache, tables, grown.totals, weights, keep, sinks=sinks, recent=recent, status=st)
        for l in range(layers):
            for r in range(n):
                for h in range(kv):
                    t = len(kept[l][r][h])
                    places = e.kept[l, r, h].tolist()
                    mine = U.evict(weights[l, r, h, :t].tolist(), keep, sinks, recent)
                    assert places == mine + [-1] * (keep - len(mine))
                    assert torch.allclose(weights[l, r, h, :t].double().cpu(), torch.tensor(given[l][r][h], dtype=torch.float64), rtol=1e-3, atol=1e-5)
                    kept[l][r][h] = [kept[l][r][h][i] for i in mine]
                    given[l][r][h] = [given[l][r][h][i] for i in mine]
        weights = e.weights.clone()
        back = block_tables(tables, e.lengths, torch.zeros_like(lengths), free, span, page, 0, held=grown.totals, status=st)
        span, lengths = back.free_range, e.lengths
        st.check_status()
        assert lengths.tolist() == [min(keep, t + 1) for t in old.tolist()]
        used = sum(-(-t // page) for t in lengths.tolist())
        assert (span[1] - span[0]).item() == pool - used


def test_captured_steps_on_another_stream():
    """Every operator in graphs of one pool that are replayed with other lengths, one of them past what was written: the eager results, bit by bit."""
    from actfold_b200.speculative import Int4Cache, attention_weights, evict_cache, read_cache_int4, tree_attention_int4, write_cache_int4

    def case(kind, seed):
        a, starts, _ = _attention_case(ls=[300, 1200, 40], dim=128, page=16, dtype=BF, tree=False, seed=seed, **KINDS[kind])
        total, heads = a["q"].shape[:2]
        kv = KINDS[kind]["kv"]
        g = torch.Generator(device="cuda").manual_seed(seed)
        a["weights"] = torch.rand(3, kv, 1300, device="cuda", generator=g)
        a["slots"] = a["tables"][1, 5].long() * 16 + torch.arange(4, device="cuda")
        a["rows"] = torch.randn(4, kv, 128, device="cuda", generator=g).to(BF)
        return a

    def step(a, cache, weights):
        args = {x: a[x] for x in ("q", "k", "v", "tables", "lengths", "starts", "mask")}
        lse = torch.empty(a["q"].shape[0], a["q"].shape[1], device="cuda")
        write_cache_int4(a["rows"], a["rows"], cache, a["slots"])
        out = tree_attention_int4(**args, cache=cache, lse=lse)
        attention_weights(a["q"], cache, a["tables"], a["lengths"], a["starts"], lse, weights)
        e = evict_cache(cache, a["tables"], a["lengths"], weights, 200, sinks=2, recent=20)
        return out, lse, *e, *read_cache_int4(cache, a["slots"])

    cases = [case(kind, 20 + i) for i, kind in enumerate(KINDS)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results, caches, sums = [], [], [], []
    pool = torch.cuda.graph_pool_handle()
    with torch.cuda.stream(side):
        for a in cases:
            caches.append(Int4Cache(a["cache"].data.clone(), BF))
            sums.append(a["weights"].clone())
            step(a, caches[-1], sums[-1])
        side.synchronize()
        for a, c, w in zip(cases, caches, sums):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, pool=pool, stream=side):
                results.append(step(a, c, w))
            graphs.append(gr)
    for ls in ([300, 1200, 40], [1, 900, 201], [0, 0, 640]):
        for a, gr, r, c, w in zip(cases, graphs, results, caches, sums):
            a["lengths"].copy_(_i32(ls))
            c.data.copy_(a["cache"].data)
            w.copy_(a["weights"])
            c2, w2 = Int4Cache(a["cache"].data.clone(), BF), a["weights"].clone()
            want = step(a, c2, w2)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                gr.replay()
            side.synchronize()
            for x, y in zip((*r, c.data, w), (*want, c2.data, w2)):
                assert torch.equal(_bits(x), _bits(y))
    torch.cuda.synchronize()


def test_calls_at_once_on_two_streams():
    """Two attentions and two evictions on streams of their own, each with its own scratch."""
    from actfold_b200.speculative import Int4Cache, evict_cache, tree_attention_int4

    cases = [_attention_case(ls=[3000, 2000, 900], dim=128, page=16, dtype=BF, tree=False, seed=30 + i, **KINDS[kind])[0] for i, kind in enumerate(("8", "128"))]
    want = [tree_attention_int4(**a) for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, (a, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(tree_attention_int4(**a))
    evicted = []
    for a, s in zip(cases, streams):
        with torch.cuda.stream(s):
            c = Int4Cache(a["cache"].data.clone(), BF)
            w = torch.arange(3000, device="cuda", dtype=torch.float32).flip(0).expand(3, 2, 3000)
            evicted.append((c, evict_cache(c, a["tables"], a["lengths"], w, 1000)))
    for s in streams:
        s.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(_bits(x), _bits(z)) for z in y)
    for c, e in evicted:
        assert e.lengths.tolist() == [1000, 1000, 900] and torch.equal(e.kept[0, 0], torch.arange(1000, device="cuda", dtype=torch.int32))


def test_empty_calls():
    from actfold_b200.speculative import Int4Cache, attention_weights, evict_cache, read_cache_int4, tree_attention_int4, write_cache_int4

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    cache = Int4Cache.empty(2, 8, 2, 64, BF)
    none = Int4Cache.empty(0, 8, 2, 64, BF)
    q, k = (torch.ones(3, h, 64, dtype=BF, device="cuda") for h in (4, 2))
    assert tree_attention_int4(q[:0], k[:0], k[:0], cache, i32(2, 1), i32(2), i32(3)).shape == (0, 4, 64)
    assert tree_attention_int4(q, k, k, cache, i32(0, 1), i32(0), i32(1)).shape == (3, 4, 64)
    for c, t in ((cache, i32(1, 0)), (none, i32(1, 2)), (cache, i32(1, 1))):  # no table entries, no pages, no cached token
        out = tree_attention_int4(q, k, k, c, t, i32(1), _i32([0, 3]))
        assert torch.equal(out, q)
    w = torch.ones(1, 2, 8, device="cuda")
    for c, t in ((cache, i32(1, 0)), (none, i32(1, 2)), (cache, i32(1, 1))):
        assert bool((attention_weights(q, c, t, i32(1), _i32([0, 3]), torch.zeros(3, 4, device="cuda"), w) == 1).all())
        e = evict_cache(c, t, i32(1), w, 4)
        assert e.lengths.tolist() == [0] and bool((e.kept == -1).all()) and not e.weights.any()
    assert evict_cache(cache, i32(0, 1), i32(0), w[:0], 4).kept.shape == (0, 2, 4)
    empty = torch.zeros(0, 2, 8, 2, 64, dtype=BF, device="cuda")
    e = evict_cache((empty, empty), i32(1, 1), _i32([9]), torch.zeros(0, 1, 2, 8, device="cuda"), 4)
    assert e.lengths.tolist() == [4] and e.kept.shape == (0, 1, 2, 4)
    write_cache_int4(k, k, none, torch.full((3,), -1, dtype=torch.int64, device="cuda"))
    assert not read_cache_int4(none, torch.full((3,), -1, dtype=torch.int64, device="cuda"))[0].any()
