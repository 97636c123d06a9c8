"""Measured cases of the operators that keep long requests in less memory: a paged key/value cache in 4 bits.

Four operators next to the 16-bit cache's: rows into and out of a 4-bit cache
(``write_cache_int4``, ``read_cache_int4``), attention of drafted trees over
it, with a sliding window and first tokens that stay visible
(``tree_attention_int4``), the attention weight that cached tokens are given
(``attention_weights``), and the eviction of those that were given least
(``evict_cache``). ``run`` computes a case in plain torch operations, or,
where ``own`` is set, through the framework.

A cached head of 8 tokens is one block of 10 * dim bytes: codes of the keys (8
rows of dim / 2 bytes), their scales and offsets (8 rows of a 16-bit pair per
32 dims), then the same of the values. Word w of a row of codes holds dims 8 w
to 8 w + 7: bits 4 i of its low half dim 8 w + 2 i, of its high half dim 8 w +
2 i + 1. With 128 dims the two halves of a row of codes are swapped in rows 2,
3, 6 and 7. A value is code * scale + offset, rounded once to the pair's type.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"
GROUP = 32  # dims that share a scale and an offset


# ---------------------------------------------------------------------------------------------- cases
def listed():
    """The head layouts are those of the two served architectures: 28 query heads over 4 key/value heads, and 32 over 32."""
    return [
        # Accepted rows of all 28 layers of a batch, and one layer's rows of long prompts, into their slots; read back, as for a step that needs 16 bits.
        dict(name="store accepted", op="store", layers=28, batch=16, keep=8, nodes=64, heads=4, dim=128, page=16, dtype="bf16", prompt=False),
        dict(name="store prompts", op="store", layers=1, batch=9, keep=1801, nodes=1801, heads=32, dim=128, page=64, dtype="bf16", prompt=True),
        # One request, one new token, a short chat so far: the smallest call, once per layer and token.
        dict(name="attention one token", op="attention", batch=1, nodes=1, least_nodes=1, length=523, least_length=523, heads=28, kv_heads=4,
             dim=128, page=16, dtype="bf16", chain=True, window=0, sinks=0),
        # A served batch decoding one token each, lengths spread as requests come and go.
        dict(name="attention batch of tokens", op="attention", batch=64, nodes=1, least_nodes=1, length=8000, least_length=90, heads=28,
             kv_heads=4, dim=128, page=64, dtype="bf16", chain=True, window=0, sinks=0),
        # Long streams behind a window, every query head with keys of its own.
        dict(name="attention window", op="attention", batch=24, nodes=1, least_nodes=1, length=30000, least_length=500, heads=32, kv_heads=32,
             dim=128, page=64, dtype="bf16", chain=True, window=4096, sinks=4),
        # Drafted trees of a batch verified over ordinary caches, every query head with keys of its own.
        dict(name="attention trees", op="attention", batch=8, nodes=64, least_nodes=20, length=4100, least_length=300, heads=32, kv_heads=32,
             dim=128, page=64, dtype="bf16", chain=False, window=0, sinks=0),
        # Drafted trees over long documents, grouped heads.
        dict(name="attention trees long", op="attention", batch=4, nodes=64, least_nodes=48, length=65500, least_length=30000, heads=28,
             kv_heads=4, dim=128, page=16, dtype="f16", chain=False, window=0, sinks=0),
        # One request's new token, and a batch's accepted tokens: the weight that they give to every cached token.
        dict(name="weights one token", op="weights", batch=1, nodes=1, length=1500, least_length=1500, heads=28, kv_heads=4, dim=128, page=16,
             dtype="bf16", held=4, window=0, sinks=0),
        dict(name="weights batch", op="weights", batch=64, nodes=4, length=8000, least_length=90, heads=28, kv_heads=4, dim=128, page=64,
             dtype="bf16", held=4, window=0, sinks=0),
        # One request over its budget, all 28 layers in 4 bits; a batch over it, a few layers in 16 bits.
        dict(name="evict one request", op="evict", layers=28, batch=1, length=4100, least_length=4100, keep=2048, heads=4, dim=128, page=16,
             dtype="bf16", held=4, sinks=4, recent=256),
        dict(name="evict batch", op="evict", layers=6, batch=16, length=4100, least_length=900, keep=1500, heads=4, dim=128, page=64,
             dtype="bf16", held=16, sinks=4, recent=100),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"] + w["flops"] / 250)
    op = rng.choice(["attention", "attention", "attention", "store", "weights", "evict"])
    case = None
    while case is None or work(case)["bytes"] + work(case)["flops"] / 250 > most[op] or _cached(case) > 4e9:
        kv, group = rng.choice([(4, 7), (32, 1), (8, 4), (2, 8), (1, 12), (5, 3)])
        dim, page, dtype = rng.choice([64, 128, 128]), rng.choice([8, 16, 32, 48, 64, 128]), rng.choice(["bf16", "f16"])
        if op == "attention":
            chain = rng.random() < 0.5
            nodes = _spread(rng, 1, 64 if chain else 256)
            length = _spread(rng, 1, 65500)
            window = _spread(rng, 1, 8000) if rng.random() < 0.4 else 0
            case = dict(op=op, batch=_spread(rng, 1, 64), nodes=nodes, least_nodes=rng.randint(1, nodes), length=length,
                        least_length=rng.randint(0, length), heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype, chain=chain,
                        window=window, sinks=rng.randint(0, 8) if window else 0)
            # The padded plain form holds a batch's scores and rows: no more than the largest listed cases'.
            t = min(length, window + case["sinks"]) if window else length
            if case["batch"] * case["heads"] * nodes * (t + nodes) > 4 * 28 * 64 * 65600 or case["batch"] * kv * dim * t > 64 * 4 * 128 * 16000:
                case = None
        elif op == "store":
            prompt = rng.random() < 0.5
            case = dict(op=op, layers=1 if prompt else _spread(rng, 1, 28), batch=_spread(rng, 1, 16),
                        keep=_spread(rng, 1, 1800) if prompt else rng.randint(1, 12), nodes=0, heads=kv, dim=dim, page=page, dtype=dtype, prompt=prompt)
            case["nodes"] = case["keep"] if prompt else case["keep"] + rng.randint(0, 60)
        elif op == "weights":
            length = _spread(rng, 1, 30000)
            window = _spread(rng, 1, 8000) if rng.random() < 0.3 else 0
            case = dict(op=op, batch=_spread(rng, 1, 64), nodes=_spread(rng, 1, 12), length=length, least_length=rng.randint(0, length),
                        heads=kv * group, kv_heads=kv, dim=dim, page=page, dtype=dtype, held=rng.choice([4, 4, 16]), window=window,
                        sinks=rng.randint(0, 8) if window else 0)
        else:
            length = _spread(rng, 10, 30000)
            keep = rng.randint(1, length + length // 4)
            sinks = min(keep, rng.randint(0, 8))
            case = dict(op=op, layers=_spread(rng, 1, 28), batch=_spread(rng, 1, 16), length=length, least_length=rng.randint(0, length), keep=keep,
                        heads=kv, dim=dim, page=page, dtype=dtype, held=rng.choice([4, 16]), sinks=sinks, recent=rng.randint(0, (keep - sinks) // 2))
    return case


def _between(low, high, count):
    """`count` whole numbers from `high` down to `low`, unevenly spread: the sizes of a batch, alike for every seed."""
    return [low + ((high - low) * ((i * 7919 + 1) % 101) + 50) // 101 if i else high for i in range(count)]


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(c):
    return _between(c["least_length"], c["length"], c["batch"])


def _nodes(c):
    return _between(c.get("least_nodes", 1), c["nodes"], c["batch"])


def _kept(c):
    """New tokens per request of a store case."""
    return _between(max(1, c["keep"] // 4), c["keep"], c["batch"])


def _cached(c):
    """Bytes of the cache that a case needs, whatever of it is read."""
    if c["op"] == "store":
        return 0
    return c.get("layers", 1) * sum(_lengths(c)) * c.get("kv_heads", c["heads"]) * c["dim"] * (4 if c.get("held") == 16 else 1.25)


def work(case):
    c, op = case, case["op"]
    held = c["dim"] * 5 // 8  # bytes of a cached key or value of one head in 4 bits
    if op == "store":
        rows = c["layers"] * sum(_kept(c)) * c["heads"]
        # Rows come in once and go out once; the cached bytes in between are written and read.
        return {"bytes": rows * (8 * c["dim"] + 4 * held), "flops": 0}
    ls = _lengths(c)
    if op == "evict":
        row = 2 * held if c["held"] == 4 else 4 * c["dim"]
        over = [t for t in ls if t > c["keep"]]
        # A token behind the first sinks moves; all but the last recent ones are looked at. What is in 4 bits is returned as values.
        moved, seen = len(over) * (c["keep"] - c["sinks"]), sum(over)
        back = c["layers"] * c["heads"] * sum(min(t, c["keep"]) for t in ls) * (row + 4 * c["dim"]) if c["held"] == 4 else 0
        return {"bytes": c["layers"] * c["heads"] * (2 * moved * row + 8 * seen + 4 * len(ls) * c["keep"]) + back, "flops": 0}
    ns = _nodes(c)
    seen = [min(t, c["window"] + c["sinks"]) if c["window"] else t for t in ls]
    rows = sum(ns) * c["heads"]
    if op == "weights":
        row = held if c["held"] == 4 else 2 * c["dim"]
        return {"bytes": sum(seen) * c["kv_heads"] * (row + 8) + rows * (2 * c["dim"] + 4),
                "flops": 2 * c["dim"] * c["heads"] * sum(n * t for n, t in zip(ns, seen))}
    mask = 0 if c["chain"] else sum(ns) * 4 * _pages(c["nodes"], 32)
    return {"bytes": 2 * sum(seen) * c["kv_heads"] * held + 4 * sum(ns) * c["kv_heads"] * c["dim"] + 4 * rows * c["dim"] + mask
            + 4 * sum(_pages(t, c["page"]) for t in seen),
            "flops": 4 * c["dim"] * c["heads"] * sum(n * (n + t) for n, t in zip(ns, seen))}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _starts(counts):
    return _ints([0] + torch.tensor(counts).cumsum(0).tolist())


def _ancestor_bits(ns, words, g):
    """Ancestor bits of random trees, each node's parent up to 32 places back, as a drafter that grows its best leaves lays them out."""
    most, b = max(ns), len(ns)
    i = torch.arange(most, device=DEV)
    back = 1 + (torch.rand(b, most, device=DEV, generator=g) * i.clamp(max=32)).long()
    jump = torch.where(i == 0, most, (i - back).clamp(min=0)).expand(b, most)
    jump = torch.cat([jump, _ints([[most]] * b, torch.int64)], 1)
    seen = torch.zeros(b, most + 1, 32 * words, dtype=torch.bool, device=DEV)
    seen[:, i, i] = True
    for _ in range(max(1, most.bit_length())):
        seen = seen | seen.gather(1, jump[..., None].expand(-1, -1, 32 * words))
        jump = jump.gather(1, jump)
    bits = (seen[:, :most].view(b, most, words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    there = i < _ints(ns)[:, None]
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)[there]


def _tables(ls, page, g):
    """Pages of a request lie scattered over the pool: (tables, pages of the pool)."""
    used = [_pages(t, page) for t in ls]
    pool, most = sum(used) + 3, max(1, max(used))
    order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    tables = torch.full((len(ls) * most,), -1, dtype=torch.int32, device=DEV)
    at = torch.cat([torch.arange(u) + i * most for i, u in enumerate(used)]).to(DEV)
    tables[at] = order[: sum(used)]
    return tables.view(len(ls), most), pool


def _blocks(outer, heads, page, dim, dtype, g):
    """Random 4-bit pages [*outer, heads, page / 8, 10 dim]: keys with a few strong channels, as rotated keys have."""
    data = torch.randint(0, 256, (*outer, heads, page // 8, 2, 5 * dim), dtype=torch.uint8, device=DEV, generator=g)
    shape = (*outer, heads, page // 8, 2, 8, dim // GROUP)
    strong = torch.where(torch.rand(heads, 1, 2, 1, dim // GROUP, device=DEV, generator=g) < 0.2, 2.0, 1.0)
    strong[:, :, 1] = 1.0
    scale = (0.2 + 0.1 * torch.rand(shape, device=DEV, generator=g)) * strong
    offset = -scale * (6 + 3 * torch.rand(shape, device=DEV, generator=g))
    data[..., 4 * dim:] = torch.stack([scale.to(dtype), offset.to(dtype)], -1).flatten(-3).view(torch.uint8)
    return data.view(*outer, heads, page // 8, 10 * dim)


def prepare(case, seed):
    c, op, g = case, case["op"], _gen(seed)
    if op == "store":
        return _prepare_store(c, g)
    dtype, dim, ls = DTYPES[c["dtype"]], c["dim"], _lengths(c)
    tables, pool = _tables(ls, c["page"], g)

    def rand(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    s = dict(op=op, tables=tables, lengths=_ints(ls), longest=max(ls), dtype=dtype, dim=dim, sinks=c["sinks"], held=c.get("held", 4))
    if op == "evict":
        outer = (c["layers"], pool)
        # Few tokens get most of the weight; some get none at all.
        w = torch.rand(c["layers"], c["batch"], c["heads"], max(ls) + 5, device=DEV, generator=g)
        s.update(weights=(w - 0.02).clamp(min=0) ** 4 * 30, keep=c["keep"], recent=c["recent"])
        if c["held"] == 4:
            s["data"] = _blocks(outer, c["heads"], c["page"], dim, dtype, g)
        else:
            s["k_cache"], s["v_cache"] = (rand(*outer, c["page"], c["heads"], dim).to(dtype) for _ in range(2))
        return s
    ns = _nodes(c)
    total, kv = sum(ns), c["kv_heads"]
    strong = torch.where(torch.rand(kv, dim, device=DEV, generator=g) < 0.04, 3.0, 1.0)
    s.update(q=rand(total, c["heads"], dim).to(dtype), starts=_starts(ns), most_nodes=max(ns), window=c["window"] or None)
    if c.get("held", 4) == 4:
        s["data"] = _blocks((pool,), kv, c["page"], dim, dtype, g)
    else:
        s["k_cache"] = (rand(pool, c["page"], kv, dim) * strong).to(dtype)
    if op == "weights":
        # The rows' logs of sums as the attention leaves them: near log(tokens) + half the scores' variance.
        s["lse"] = torch.log(s["lengths"].float() + 1).repeat_interleave(s["starts"][1:] - s["starts"][:-1], output_size=total)[:, None] \
            + 1.5 + 0.5 * rand(total, c["heads"])
        s["weights"] = torch.rand(c["batch"], kv, max(ls) + 3, device=DEV, generator=g)
        return s
    s.update(k=(rand(total, kv, dim) * strong).to(dtype), v=rand(total, kv, dim).to(dtype),
             mask=None if c["chain"] else _ancestor_bits(ns, _pages(c["nodes"], 32), g))
    return s


def _prepare_store(c, g):
    """A prompt's rows come packed, with a slot each; the accepted rows of a tree come by their numbers, -1 behind the last one of a request."""
    dtype, kept = DTYPES[c["dtype"]], _kept(c)
    page, b = c["page"], c["batch"]
    old = [17 + 31 * i for i in range(b)]
    pages = sum(_pages(o + n, page) for o, n in zip(old, kept))
    order = torch.randperm(pages, device=DEV, generator=g)
    first = torch.tensor([0] + [_pages(o + n, page) for o, n in zip(old, kept)]).cumsum(0)[:-1].tolist()
    position = torch.cat([first[i] * page + o + torch.arange(n) for i, (o, n) in enumerate(zip(old, kept))]).to(DEV)
    slots = order[position // page] * page + position % page
    if c["prompt"]:
        rows, total = None, sum(kept)
    else:
        total = c["nodes"] * b
        pick = torch.rand(b, c["nodes"], device=DEV, generator=g).argsort(1)[:, : c["keep"]].sort(1).values
        live = torch.arange(c["keep"], device=DEV)[None] < _ints(kept)[:, None]
        rows = torch.where(live, pick + torch.arange(b, device=DEV)[:, None] * c["nodes"], -1).to(torch.int32)
        at = torch.full((b, c["keep"]), -1, dtype=torch.int64, device=DEV)
        at[live] = slots
        slots = at
    k, v = (torch.randn(c["layers"], total, c["heads"], c["dim"], device=DEV, generator=g).to(dtype) for _ in range(2))
    k[..., 5] *= 4  # one strong channel
    data = torch.randint(0, 256, (c["layers"], pages, c["heads"], page // 8, 10 * c["dim"]), dtype=torch.uint8, device=DEV, generator=g)
    return dict(op="store", k=k, v=v, data=data, slots=slots, rows=rows, dtype=dtype)


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attention": _plain_attention, "weights": _plain_weights, "evict": _plain_evict}[state["op"]](state)


def _own(s):
    from actfold_b200 import speculative as spec

    if s["op"] == "store":
        cache = spec.Int4Cache(s["data"], s["dtype"])
        spec.write_cache_int4(s["k"], s["v"], cache, s["slots"], rows=s["rows"])
        k, v = spec.read_cache_int4(cache, s["slots"])
        return {"k": k, "v": v}
    if s["op"] == "attention":
        cache = spec.Int4Cache(s["data"], s["dtype"])
        mask = s["mask"]
        if mask is None and s["sinks"] and s["window"] < s["most_nodes"]:
            mask = _last_nodes(s)  # the first tokens that stay are the prefix's here; without bits a chain's own first ones would stay too
        return {"out": spec.tree_attention_int4(s["q"], s["k"], s["v"], cache, s["tables"], s["lengths"], s["starts"], mask,
                                                window=s["window"], sinks=s["sinks"])}
    if s["op"] == "weights":
        cache = spec.Int4Cache(s["data"], s["dtype"]) if s["held"] == 4 else s["k_cache"]
        spec.attention_weights(s["q"], cache, s["tables"], s["lengths"], s["starts"], s["lse"], s["weights"], window=s["window"], sinks=s["sinks"])
        return {"weights": s["weights"]}
    cache = spec.Int4Cache(s["data"], s["dtype"]) if s["held"] == 4 else (s["k_cache"], s["v_cache"])
    r = spec.evict_cache(cache, s["tables"], s["lengths"], s["weights"], s["keep"], sinks=s["sinks"], recent=s["recent"])
    if s["held"] == 16:
        return {"kept": r.kept, "lengths": r.lengths, "weights": r.weights, "k": s["k_cache"], "v": s["v_cache"]}
    k, v = spec.read_cache_int4(cache, _kept_slots(s))
    return {"kept": r.kept, "lengths": r.lengths, "weights": r.weights, "k": k, "v": v}


def _last_nodes(s):
    """Bits of the last `window` nodes of its chain for every node."""
    starts, total = s["starts"].long(), s["q"].shape[0]
    i = torch.arange(total, device=DEV) - starts[:-1].repeat_interleave(starts[1:] - starts[:-1], output_size=total)
    j = torch.arange(32 * _pages(s["most_nodes"], 32), device=DEV)
    sees = (j <= i[:, None]) & (j > i[:, None] - s["window"])
    bits = (sees.view(total, -1, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)


def _kept_slots(s):
    """Slots of the first `keep` places of every request, -1 behind its last token."""
    place = torch.arange(min(s["keep"], s["longest"]), device=DEV)
    page = s["data"].shape[-2] * 8
    slots = s["tables"].long()[:, place // page] * page + place % page
    return torch.where(place < s["lengths"][:, None], slots, -1)


def _values(data, dtype, slots):
    """Keys and values [..., 2, n.., heads, dim] in fp32 that the 4-bit pages [..., pages, heads, page / 8, 10 dim] hold at `slots`."""
    *outer, pages, heads, blocks, size = data.shape
    dim = size // 10
    rows = data.view(*outer, pages, heads, blocks, 2, 5 * dim)
    flat = slots.reshape(-1)
    block, r = flat // 8, flat % 8
    rows = rows[..., block // blocks, :, block % blocks, :, :]  # advanced indexes apart: their dimension comes first
    rows = rows.view(flat.numel(), *outer, heads, 2, 5 * dim)
    lead = (flat.numel(),) + (1,) * (len(outer) + 2)
    codes = rows[..., : 4 * dim].view(*rows.shape[:-1], 8, dim // 2)
    codes = codes.gather(-2, r.view(*lead, 1, 1).expand(*rows.shape[:-1], 1, dim // 2)).squeeze(-2)
    pairs = rows[..., 4 * dim:].view(*rows.shape[:-1], 8, dim // 8)
    pairs = pairs.gather(-2, r.view(*lead, 1, 1).expand(*rows.shape[:-1], 1, dim // 8)).squeeze(-2).contiguous().view(dtype)
    if dim == 128:
        swapped = ((r // 2) % 2 == 1).view(*lead, 1)
        codes = torch.where(swapped, codes.roll(dim // 4, -1), codes)
    # Bytes 0 to 3 of a word: nibbles of dims (0, 2), (4, 6), (1, 3), (5, 7).
    nibbles = torch.stack([codes & 15, codes >> 4], -1).view(*codes.shape[:-1], dim // 8, 2, 4).transpose(-1, -2).reshape(*codes.shape[:-1], dim)
    scale, offset = (pairs.float().view(*pairs.shape[:-1], dim // GROUP, 2)[..., i].repeat_interleave(GROUP, -1) for i in (0, 1))
    x = (nibbles.float() * scale + offset).to(dtype).float()
    return x.movedim(0, len(outer)).movedim(-2, 0).reshape(2, *outer, *slots.shape, heads, dim)


def _plain_store(s):
    """Rows into codes, scales and offsets, these into their slots' bytes, and the slots' bytes back into values."""
    data, dtype, slots = s["data"], s["dtype"], s["slots"]
    layers, pages, heads, blocks, size = data.shape
    dim = size // 10
    rows = torch.arange(slots.numel(), device=DEV) if s["rows"] is None else s["rows"].reshape(-1).clamp(min=0)
    live = slots.reshape(-1) >= 0
    at = slots.reshape(-1).clamp(min=0)
    x = torch.stack([s["k"][:, rows], s["v"][:, rows]]).float().view(2, layers, -1, heads, dim // GROUP, GROUP)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(dtype).float()
    # (in 64 bits: a quotient next to a border between two codes)
    code = torch.where(scale > 0, ((x.double() - low) / torch.where(scale > 0, scale, 1.0)).round().clamp(0, 15), 0.0).to(torch.uint8)
    pairs = torch.cat([scale, low], -1).to(dtype).view(2, layers, -1, heads, dim // GROUP * 2).view(torch.uint8)
    code = code.view(2, layers, -1, heads, dim // 8, 4, 2).transpose(-1, -2).reshape(2, layers, -1, heads, dim // 2, 2)
    code = code[..., 0] | (code[..., 1] << 4)
    block, r = at // 8, at % 8
    if dim == 128:
        code = torch.where(((r // 2) % 2 == 1).view(-1, 1, 1), code.roll(dim // 4, -1), code)
    keep = live.nonzero()[:, 0] if s["rows"] is not None else slice(None)
    block, r = block[keep], r[keep]
    view = data.view(layers, pages, heads, blocks, 2, 5 * dim)
    for i in range(2):
        part = view[..., i, :]
        rows_of, pairs_of = part[..., : 4 * dim].unflatten(-1, (8, dim // 2)), part[..., 4 * dim:].unflatten(-1, (8, dim // 8))
        rows_of[:, block // blocks, :, block % blocks, r] = code[i][:, keep].movedim(1, 0)
        pairs_of[:, block // blocks, :, block % blocks, r] = pairs[i][:, keep].movedim(1, 0)
    k, v = _values(data, dtype, slots.clamp(min=0))
    there = (slots >= 0)[..., None, None]
    return {"k": torch.where(there, k, 0.0).to(dtype), "v": torch.where(there, v, 0.0).to(dtype)}


def _places(s):
    """Places [b, t] that any row of a request may see and whether they are ones: all, or the sinks and a window's."""
    lengths, longest = s["lengths"].long()[:, None], s["longest"]
    if s["window"] is None or s["window"] + s["sinks"] >= longest:
        place = torch.arange(longest, device=DEV).expand(lengths.shape[0], longest)
        return place, place < lengths
    first = (lengths - s["window"]).clamp(min=s["sinks"])
    place = torch.cat([torch.arange(s["sinks"], device=DEV).expand(lengths.shape[0], s["sinks"]), first + torch.arange(s["window"], device=DEV)], 1)
    return place, place < lengths


def _slots(s, place, page):
    return s["tables"].long().gather(1, (place // page).clamp(max=s["tables"].shape[1] - 1)).clamp(min=0) * page + place % page


def _rows(s):
    """Every request padded to the most nodes: (row of a node [b, n], whether it is one, node numbers)."""
    starts = s["starts"].long()
    node = torch.arange(s["most_nodes"], device=DEV)
    return (starts[:-1, None] + node).clamp(max=s["q"].shape[0] - 1), node < (starts[1:] - starts[:-1])[:, None], node


def _in_window(s, place, count):
    """Places [b, 1, t] that nodes with `count` [b, n] visible nodes of their own tree see."""
    if s["window"] is None:
        return True
    first = s["lengths"].long()[:, None] - (s["window"] - count).clamp(min=0)
    return (place[:, None] >= first[..., None]) | (place[:, None] < s["sinks"])


def _plain_attention(s):
    """Every request padded to the longest: out = softmax(q k^T / sqrt(dim)) v over the cached keys and the tree's visible ones."""
    q, data = s["q"], s["data"]
    total, heads, dim = q.shape
    kv = data.shape[1]
    row, there, node = _rows(s)
    b, n = row.shape
    place, cached = _places(s)
    t = place.shape[1]
    k, v = _values(data, s["dtype"], _slots(s, place, data.shape[2] * 8))
    k, v = torch.cat([k, s["k"][row].float()], 1), torch.cat([v, s["v"][row].float()], 1)  # [b, t + n, kv, dim]
    if s["mask"] is None:
        sees = (node <= node[:, None]).expand(b, n, n)
        if s["window"] is not None:
            sees = sees & (node > node[:, None] - s["window"])
    else:
        sees = ((s["mask"][row][..., node // 32] >> (node % 32)) & 1).bool()  # [b, n, n]
    sees = sees & there[:, None]
    sees = torch.cat([(cached[:, None] & _in_window(s, place, sees.sum(-1))).expand(b, n, t), sees], 2)
    x = q[row].float().view(b, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)  # rows: head of the group, node
    scores = (x @ k.permute(0, 2, 3, 1) * dim ** -0.5).view(b, kv, heads // kv, n, t + n)
    scores = torch.where(sees[:, None, None], scores, -math.inf)
    del k
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total_p = scores.sum(-1, keepdim=True)
    out = scores.view(b, kv, -1, t + n) @ v.permute(0, 2, 1, 3)
    out = out.view(b, kv, -1, n, dim) / torch.where(total_p > 0, total_p, 1.0)
    return {"out": out.permute(0, 3, 1, 2, 4)[there].reshape(total, heads, dim).to(q.dtype)}


def _plain_weights(s):
    """weights[b, h, p] += the probabilities that all rows of the request and all query heads of the group give to place p."""
    q, weights = s["q"], s["weights"]
    total, heads, dim = q.shape
    kv = weights.shape[1]
    row, there, node = _rows(s)
    b, n = row.shape
    place, cached = _places(s)
    if s["held"] == 4:
        k = _values(s["data"], s["dtype"], _slots(s, place, s["data"].shape[2] * 8))[0]
    else:
        k = s["k_cache"].flatten(0, 1)[_slots(s, place, s["k_cache"].shape[1])].float()
    x = q[row].float().view(b, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)
    scores = (x @ k.permute(0, 2, 3, 1) * dim ** -0.5).view(b, kv, heads // kv, n, -1)
    scores -= s["lse"][row].view(b, n, kv, heads // kv).permute(0, 2, 3, 1)[..., None]
    count = node + 1 if s["window"] is None else (node + 1).clamp(max=s["window"])
    sees = cached[:, None] & there[..., None] & _in_window(s, place, count.expand(b, n))
    given = torch.where(sees[:, None, None], scores.exp_(), 0.0).sum((2, 3))
    weights.scatter_add_(2, place[:, None].expand(b, kv, -1).clamp(max=weights.shape[2] - 1), given)
    return {"weights": weights}


def _plain_evict(s):
    """Of every request, layer and head with more than `keep` tokens: the first, the last and the heaviest between stay, moved to the front in order."""
    weights, keep, lengths = s["weights"], s["keep"], s["lengths"].long()
    layers, b, heads, width = weights.shape
    place = torch.arange(width, device=DEV)
    there = place < lengths[:, None]
    always = there & ((place < s["sinks"]) | (place >= lengths[:, None] - s["recent"]))
    order = torch.where(always[:, None], math.inf, torch.where(there[:, None], weights, -math.inf)).sort(dim=-1, descending=True, stable=True).indices
    best = order[..., :keep].sort(-1).values
    short = (lengths <= keep)[:, None, None]
    number = torch.arange(best.shape[-1], device=DEV)
    kept = torch.where(short, number, best)
    new = lengths.clamp(max=keep)
    live = number < new[:, None, None]
    out = torch.zeros_like(weights)
    out[..., : kept.shape[-1]] = torch.where(live, weights.gather(-1, kept), 0.0)
    result = torch.full((layers, b, heads, keep), -1, dtype=torch.int32, device=DEV)
    result[..., : kept.shape[-1]] = torch.where(live, kept, -1).to(torch.int32)
    move = live & ~short
    l, r, h, d = torch.nonzero(move.expand_as(kept), as_tuple=True)
    tables, src = s["tables"].long(), kept[l, r, h, d]
    if s["held"] == 16:
        page = s["k_cache"].shape[2]
        for cache in (s["k_cache"], s["v_cache"]):
            cache[l, tables[r, d // page], d % page, h] = cache[l, tables[r, src // page], src % page, h]
        return {"kept": result, "lengths": new.to(torch.int32), "weights": out, "k": s["k_cache"], "v": s["v_cache"]}
    dim, page = s["dim"], s["data"].shape[-2] * 8
    view = s["data"].unflatten(-1, (2, 5 * dim))
    for i in range(2):
        part = view[..., i, :]
        rows_of, pairs_of = part[..., : 4 * dim].unflatten(-1, (8, dim // 2)), part[..., 4 * dim:].unflatten(-1, (8, dim // 8))
        codes = rows_of[l, tables[r, src // page], h, src % page // 8, src % 8]
        pairs = pairs_of[l, tables[r, src // page], h, src % page // 8, src % 8]
        if dim == 128:
            codes = torch.where((src // 2 % 2 != d // 2 % 2)[:, None], codes.roll(dim // 4, -1), codes)
        rows_of[l, tables[r, d // page], h, d % page // 8, d % 8] = codes
        pairs_of[l, tables[r, d // page], h, d % page // 8, d % 8] = pairs
    slots = _kept_slots(s)
    k, v = _values(s["data"], s["dtype"], slots.clamp(min=0))
    there = (slots >= 0)[..., None, None]
    return {"kept": result, "lengths": new.to(torch.int32), "weights": out, "k": torch.where(there, k, 0.0).to(s["dtype"]),
            "v": torch.where(there, v, 0.0).to(s["dtype"])}


# ---------------------------------------------------------------------------------------------- 64 bits
def _decoded(data, dtype):
    """All rows of 4-bit pages [pages, heads, page / 8, 10 dim] in 64 bits: [2, pages * page, heads, dim], dim by dim from the layout."""
    pages, heads, blocks, size = data.shape
    dim = size // 10
    parts = data.reshape(pages, heads, blocks, 2, 5 * dim)
    words = parts[..., : 4 * dim].contiguous().view(torch.int32).view(pages, heads, blocks, 2, 8, dim // 8)
    pairs = parts[..., 4 * dim:].contiguous().view(dtype).view(pages, heads, blocks, 2, 8, dim // GROUP, 2).double()
    out = torch.empty(pages, heads, blocks, 2, 8, dim, dtype=torch.float64, device=data.device)
    for r in range(8):
        for d in range(dim):
            w = d // 8
            if dim == 128 and r in (2, 3, 6, 7):
                w = (w + dim // 16) % (dim // 8)
            bit = 4 * (d % 8 // 2) + 16 * (d % 2)
            code = (words[..., r, w] >> bit) & 15
            out[..., r, d] = code * pairs[..., r, d // GROUP, 0] + pairs[..., r, d // GROUP, 1]
    return out.to(dtype).double().permute(3, 0, 2, 4, 1, 5).reshape(2, pages * blocks * 8, heads, dim)


def exact(case, seed):
    """Request by request in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "store":
        k, v = (_exact_rows(x, s, c) for x in (s["k"], s["v"]))
        return {"k": k, "v": v}
    if c["op"] == "evict":
        return _exact_evict(c, s)
    group, dim, page = c["heads"] // c["kv_heads"], c["dim"], c["page"]
    edges, lengths = s["starts"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if c["op"] == "weights" else None
    for r, t in enumerate(lengths):
        lo, hi = edges[r], edges[r + 1]
        n, pages = hi - lo, s["tables"][r, : _pages(t, page)].long()
        if s["held"] == 4:
            k, v = _decoded(s["data"][pages], s["dtype"])[:, :t] if t else s["q"].new_zeros(2, 0, c["kv_heads"], dim).double()
        else:
            k = s["k_cache"][pages].flatten(0, 1)[:t].double()
        tree = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        if c["op"] == "attention" and s["mask"] is not None:
            words = s["mask"][lo:hi].long() & 0xFFFFFFFF
            tree = torch.stack([(words[:, j // 32] >> (j % 32)) & 1 for j in range(n)], 1) == 1
        elif c["window"]:
            tree = tree.triu(1 - c["window"])
        prefix = torch.ones(n, t, dtype=torch.bool, device=DEV)
        if c["window"]:
            for i, count in enumerate(tree.sum(1).tolist()):
                prefix[i, c["sinks"]: max(c["sinks"], t - max(0, c["window"] - count))] = False
        for h in range(c["heads"]):
            x = s["q"][lo:hi, h].double()
            if weights is not None:
                p = torch.exp(x @ k[:, h // group].T / math.sqrt(dim) - s["lse"][lo:hi, h, None].double())
                weights[r, h // group, :t] += torch.where(prefix, p, 0.0).sum(0)
                continue
            keys = torch.cat([k[:, h // group], s["k"][lo:hi, h // group].double()])
            scores = (x @ keys.T / math.sqrt(dim)).masked_fill(~torch.cat([prefix, tree], 1), -math.inf)
            out[lo:hi, h] = torch.softmax(scores, -1) @ torch.cat([v[:, h // group], s["v"][lo:hi, h // group].double()])
    return {"out": out} if weights is None else {"weights": weights}


def _exact_rows(x, s, c):
    """What 4 bits leave of the rows that go into slots; 0 where there is no slot."""
    slots = s["slots"]
    rows = torch.arange(slots.numel(), device=DEV).view(slots.shape) if s["rows"] is None else s["rows"].long()
    parts = x[:, rows.clamp(min=0)].double().unflatten(-1, (-1, GROUP))
    offset = parts.min(-1, keepdim=True).values
    scale = ((parts.max(-1, keepdim=True).values - offset) / 15).to(s["dtype"]).double()
    code = torch.clamp(torch.round((parts - offset) / scale), 0, 15).nan_to_num(0.0)
    values = (code * scale + offset).to(s["dtype"]).double().flatten(-2)
    return values * (slots >= 0)[None, ..., None, None]


def _exact_evict(c, s):
    page, keep = c["page"], c["keep"]
    lengths = s["lengths"].tolist()
    new = s["weights"].double()
    shown = min(keep, s["longest"])
    if c["held"] == 16:
        kv = [s["k_cache"].double(), s["v_cache"].double()]
    else:
        kv = [torch.zeros(c["layers"], c["batch"], shown, c["heads"], c["dim"], dtype=torch.float64, device=DEV) for _ in range(2)]
    for l in range(c["layers"]):
        for r, t in enumerate(lengths):
            entries = s["tables"][r, : _pages(t, page)].long()
            rows = None if c["held"] == 16 else _decoded(s["data"][l][entries], s["dtype"]) if t else torch.zeros(2, 0, c["heads"], c["dim"], device=DEV).double()
            place = torch.arange(t, device=DEV)
            new[l, r, :, t:] = 0
            for h in range(c["heads"]):
                chosen = place
                if t > keep:
                    w = s["weights"][l, r, h, :t].double()
                    w[: c["sinks"]] = math.inf
                    w[t - c["recent"]:] = math.inf
                    chosen = torch.argsort(-w, stable=True)[:keep].sort().values
                    new[l, r, h, :t] = torch.cat([s["weights"][l, r, h, chosen].double(), torch.zeros(t - keep, device=DEV, dtype=torch.float64)])
                m = chosen.numel()
                if c["held"] == 4:
                    for x in range(2):
                        kv[x][l, r, :m, h] = rows[x][chosen, h]
                elif t > keep:
                    for full in kv:
                        full[l, entries[place[:m] // page], place[:m] % page, h] = full[l, entries[chosen // page], chosen % page, h].clone()
    return {"kept": None, "lengths": None, "weights": new, "k": kv[0], "v": kv[1]}
