"""Measured cases of the tree verification operators over a paged key/value cache.

Five operators of one serving step: ``block_tables`` (pages and slots from
request lengths), ``tree_masks`` (ancestor bits and positions of drafted
trees), ``tree_attention`` (drafted nodes over the cached prefix and their own
tree), ``accept_tree`` (the longest path the target model agrees with) and
``write_cache`` (key/value rows into their slots). ``run`` computes a case in
plain torch operations, or, where ``own`` is set, through the framework.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------- cases
def listed():
    """The head layouts are those of the two served architectures: 28 query heads over 4 key/value heads, and 32 over 32."""
    return [
        # One request, one new token, a short chat so far: the smallest call, once per layer and token.
        dict(name="attention one token", op="attention", batch=1, nodes=1, least_nodes=1, length=523, least_length=523, heads=28, kv_heads=4,
             dim=128, page=16, dtype="bf16", chain=True),
        # A served batch decoding one token each, lengths spread as requests come and go.
        dict(name="attention batch of tokens", op="attention", batch=64, nodes=1, least_nodes=1, length=8000, least_length=90, heads=28,
             kv_heads=4, dim=128, page=64, dtype="bf16", chain=True),
        # Drafted trees of a batch verified over ordinary caches, every query head with keys of its own.
        dict(name="attention trees", op="attention", batch=8, nodes=64, least_nodes=20, length=4100, least_length=300, heads=32, kv_heads=32,
             dim=128, page=64, dtype="bf16", chain=False),
        # Drafted trees over long documents, grouped heads.
        dict(name="attention trees long", op="attention", batch=4, nodes=64, least_nodes=48, length=65500, least_length=30000, heads=28,
             kv_heads=4, dim=128, page=16, dtype="f16", chain=False),
        # One request's tree of a usual drafter, and a batch of large trees.
        dict(name="masks one tree", op="masks", batch=1, nodes=26, least_nodes=26, branch=4),
        dict(name="masks large trees", op="masks", batch=128, nodes=500, least_nodes=60, branch=6),
        # Acceptance for one request, and for a large batch.
        dict(name="accept one tree", op="accept", batch=1, nodes=26, least_nodes=26, branch=4, keep=6, agree=0.7),
        dict(name="accept batch", op="accept", batch=256, nodes=250, least_nodes=30, branch=4, keep=12, agree=0.8),
        # A small batch in which every request keeps a few tokens; a large one with prompts coming in and requests that end.
        dict(name="tables small batch", op="tables", batch=5, length=1500, grow=6, page=16, ended=0.0, prompts=0.0),
        dict(name="tables large batch", op="tables", batch=1000, length=6000, grow=9, page=32, ended=0.05, prompts=0.04),
        # Accepted rows of all 28 layers of a batch into their slots; and one layer's rows of long prompts.
        dict(name="write accepted", op="write", layers=28, batch=16, keep=8, nodes=64, heads=4, dim=128, page=16, dtype="bf16", prompt=False),
        dict(name="write prompts", op="write", layers=1, batch=9, keep=1801, nodes=1801, heads=32, dim=128, page=64, dtype="bf16", prompt=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"] + w["flops"] / 250)
    op = rng.choice(["attention", "attention", "attention", "masks", "accept", "tables", "write"])
    case = None
    while case is None or work(case)["bytes"] + work(case)["flops"] / 250 > most[op]:
        if op == "attention":
            chain = rng.random() < 0.4
            nodes = _spread(rng, 1, 64 if chain else 256)
            length = _spread(rng, 1, 65500)
            kv, group = rng.choice([(4, 7), (32, 1), (8, 4), (2, 8), (1, 12), (5, 3)])
            case = dict(op=op, batch=_spread(rng, 1, 64), nodes=nodes, least_nodes=rng.randint(1, nodes), length=length,
                        least_length=rng.randint(0, length), heads=kv * group, kv_heads=kv, dim=rng.choice([64, 128, 128]),
                        page=rng.choice([16, 32, 48, 64, 128]), dtype=rng.choice(["bf16", "f16"]), chain=chain)
            # The padded plain form holds a batch's scores: no larger than the largest listed case's.
            if case["batch"] * case["heads"] * nodes * (length + nodes) > 4 * 28 * 64 * 65600:
                case = None
        elif op == "masks":
            nodes = _spread(rng, 1, 500)
            case = dict(op=op, batch=_spread(rng, 1, 128), nodes=nodes, least_nodes=rng.randint(1, nodes), branch=rng.randint(1, 8))
        elif op == "accept":
            nodes = _spread(rng, 1, 250)
            case = dict(op=op, batch=_spread(rng, 1, 256), nodes=nodes, least_nodes=rng.randint(1, nodes), branch=rng.randint(1, 8),
                        keep=rng.randint(1, 16), agree=rng.choice([0.3, 0.7, 0.95]))
        elif op == "tables":
            case = dict(op=op, batch=_spread(rng, 1, 1000), length=_spread(rng, 10, 6000), grow=rng.randint(1, 16),
                        page=rng.choice([8, 16, 32, 64, 100]), ended=rng.choice([0.0, 0.1]), prompts=rng.choice([0.0, 0.04]))
        else:
            prompt = rng.random() < 0.5
            case = dict(op=op, layers=1 if prompt else _spread(rng, 1, 28), batch=_spread(rng, 1, 16),
                        keep=_spread(rng, 1, 1800) if prompt else rng.randint(1, 12), nodes=0, heads=rng.choice([1, 4, 8, 32]),
                        dim=rng.choice([64, 128]), page=rng.choice([16, 48, 64]), dtype=rng.choice(["bf16", "f16", "f32"]), prompt=prompt)
            case["nodes"] = case["keep"] if prompt else case["keep"] + rng.randint(0, 60)
    return case


def _between(low, high, count):
    """`count` whole numbers from `high` down to `low`, unevenly spread: the sizes of a batch, alike for every seed."""
    return [low + ((high - low) * ((i * 7919 + 1) % 101) + 50) // 101 if i else high for i in range(count)]


def _tokens(c):
    """New tokens per request of a block table case: some requests bring a prompt."""
    return [c["grow"] * (i * 37 % 5) // 4 if i % 25 >= 25 * c["prompts"] else c["length"] // 3 + i % 50 for i in range(c["batch"])]


def _lengths(c):
    """(tokens the tables hold pages for, tokens that are kept) per request of a block table case."""
    held = _between(c["length"] // 20, c["length"], c["batch"])
    kept = [0 if i % 20 < 20 * c["ended"] else max(0, h - i % 7) for i, h in enumerate(held)]
    prompt = [i % 25 < 25 * c["prompts"] for i in range(c["batch"])]
    return [0 if p else h for p, h in zip(prompt, held)], [0 if p else k for p, k in zip(prompt, kept)]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    c, op = case, case["op"]
    if op == "attention":
        size = 2
        ns, ls = _between(c["least_nodes"], c["nodes"], c["batch"]), _between(c["least_length"], c["length"], c["batch"])
        keys = sum(n + t for n, t in zip(ns, ls))
        mask = 0 if c["chain"] else sum(ns) * 4 * -(-c["nodes"] // 32)
        rows = sum(ns) * c["heads"]
        return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * size + 2 * rows * c["dim"] * size + mask + 4 * sum(_pages(t, c["page"]) for t in ls),
                "flops": 4 * c["dim"] * c["heads"] * sum(n * (n + t) for n, t in zip(ns, ls))}
    if op in ("masks", "accept"):
        n = sum(_between(c["least_nodes"], c["nodes"], c["batch"]))
        if op == "masks":
            return {"bytes": 8 * n + 4 * n * -(-c["nodes"] // 32) + 8 * c["batch"], "flops": n}
        return {"bytes": 20 * n + c["batch"] * (4 * c["keep"] + 28), "flops": n}
    if op == "tables":
        held, kept = _lengths(c)
        grow = _tokens(c)
        moved = sum(abs(_pages(k + g, c["page"]) - _pages(h, c["page"])) for h, k, g in zip(held, kept, grow))
        return {"bytes": 8 * moved + 8 * sum(grow) + 24 * c["batch"], "flops": sum(grow)}
    rows = c["layers"] * _rows(c)
    return {"bytes": 4 * rows * c["heads"] * c["dim"] * (4 if c["dtype"] == "f32" else 2), "flops": 0}


def _rows(c):
    return sum(_kept(c))


def _kept(c):
    return _between(max(1, c["keep"] // 4), c["keep"], c["batch"])


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _starts(counts):
    return _ints([0] + torch.tensor(counts).cumsum(0).tolist())


def _trees(ns, branch, g):
    """Parents of random trees, each before its children: -1, or a node at most `branch` * 8 places back, as a drafter that
    grows its best leaves lays them out."""
    i = torch.cat([torch.arange(n) for n in ns]).to(DEV)
    back = 1 + (torch.rand(i.numel(), device=DEV, generator=g) * torch.clamp(i, max=8 * branch)).long()
    return torch.where(i == 0, -1, torch.clamp(i - back, min=0)).to(torch.int32)


def _ancestor_bits(parents, starts, words):
    """Random states need masks before the operator under test makes any: the plain form's."""
    return _plain_masks(dict(parents=parents, starts=starts, words=words, base=torch.zeros_like(starts[1:])))["mask"]


def prepare(case, seed):
    c, op, g = case, case["op"], _gen(seed)
    if op == "attention":
        return _prepare_attention(c, g)
    if op in ("masks", "accept"):
        ns = _between(c["least_nodes"], c["nodes"], c["batch"])
        s = dict(op=op, batch=c["batch"], starts=_starts(ns), parents=_trees(ns, c["branch"], g), words=-(-c["nodes"] // 32),
                 base=torch.randint(0, 5000, (c["batch"],), device=DEV, generator=g, dtype=torch.int32))
        if op == "accept":
            # A drafted token agrees with the target model's choice after its parent with probability `agree`, else it is another.
            total = sum(ns)
            s["keep"] = c["keep"]
            s["targets"] = torch.randint(0, 152064, (total,), device=DEV, generator=g)
            s["root_targets"] = torch.randint(0, 152064, (c["batch"],), device=DEV, generator=g)
            of = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), _ints(ns, torch.int64), output_size=total)
            first = s["starts"].long()[of]
            up = torch.where(s["parents"] < 0, s["root_targets"][of], s["targets"][first + s["parents"].long().clamp(min=0)])
            agree = torch.rand(total, device=DEV, generator=g) < c["agree"]
            s["tokens"] = torch.where(agree, up, torch.randint(0, 152064, (total,), device=DEV, generator=g))
        return s
    if op == "tables":
        held, kept = _lengths(c)
        grow = _tokens(c)
        most = max(_pages(max(h, k + n), c["page"]) for h, k, n in zip(held, kept, grow)) + 3
        used = [_pages(h, c["page"]) for h in held]
        need = sum(max(0, _pages(k + n, c["page"]) - u) for k, n, u in zip(kept, grow, used))
        pool = sum(used) + need + 50
        order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
        at = torch.cat([torch.arange(u) + i * most for i, u in enumerate(used)]).to(DEV) if sum(used) else torch.zeros(0, dtype=torch.int64, device=DEV)
        tables = torch.full((c["batch"] * most,), -1, dtype=torch.int32, device=DEV)
        tables[at] = order[: sum(used)]
        head = int(torch.randint(0, 5 * pool, (1,), device=DEV, generator=g))
        free = torch.full((pool,), -1, dtype=torch.int32, device=DEV)
        count = pool - sum(used)
        free[(head + torch.arange(count, device=DEV)) % pool] = order[sum(used):]
        return dict(op=op, tables=tables.view(c["batch"], most), held=_ints(held), lengths=_ints(kept), grow=_ints(grow), free=free,
                    free_range=_ints([head, head + count], torch.int64), page=c["page"], capacity=sum(grow) + 8)
    return _prepare_write(c, g)


def _prepare_attention(c, g):
    """Keys have a few strong channels, as rotated keys have; pages of a request lie scattered over the pool."""
    ns, ls = _between(c["least_nodes"], c["nodes"], c["batch"]), _between(c["least_length"], c["length"], c["batch"])
    dtype, page = DTYPES[c["dtype"]], c["page"]
    used = [_pages(t, page) for t in ls]
    pool, most = sum(used) + 3, max(1, max(used))
    order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    tables = torch.full((c["batch"] * most,), -1, dtype=torch.int32, device=DEV)
    at = torch.cat([torch.arange(u) + i * most for i, u in enumerate(used)]).to(DEV)
    tables[at] = order[: sum(used)]
    strong = torch.where(torch.rand(c["kv_heads"], c["dim"], device=DEV, generator=g) < 0.04, 3.0, 1.0)

    def rand(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    total, words = sum(ns), -(-c["nodes"] // 32)
    starts = _starts(ns)
    mask = None if c["chain"] else _ancestor_bits(_trees(ns, 4, g), starts, words)
    return dict(op="attention", q=rand(total, c["heads"], c["dim"]).to(dtype), k=(rand(total, c["kv_heads"], c["dim"]) * strong).to(dtype),
                v=rand(total, c["kv_heads"], c["dim"]).to(dtype), k_cache=(rand(pool, page, c["kv_heads"], c["dim"]) * strong).to(dtype),
                v_cache=rand(pool, page, c["kv_heads"], c["dim"]).to(dtype), tables=tables.view(c["batch"], most), lengths=_ints(ls),
                starts=starts, mask=mask, longest=max(ls), most_nodes=c["nodes"])


def _prepare_write(c, g):
    """The pool has one page more than is handed out: a place for rows that go nowhere. A prompt's rows come packed, with a slot each; the accepted
    rows of a tree come by their numbers, -1 behind the last one of a request."""
    dtype, kept = DTYPES[c["dtype"]], _kept(c)
    page, b = c["page"], c["batch"]
    old = [17 + 31 * i for i in range(b)]
    pages = sum(_pages(o + n, page) for o, n in zip(old, kept))
    order = torch.randperm(pages, device=DEV, generator=g)
    first = torch.tensor([0] + [_pages(o + n, page) for o, n in zip(old, kept)]).cumsum(0)[:-1].tolist()
    position = torch.cat([first[i] * page + o + torch.arange(n) for i, (o, n) in enumerate(zip(old, kept))]).to(DEV)
    slots = order[position // page] * page + position % page
    shape = (c["layers"], pages + 1, page, c["heads"], c["dim"])
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
    k_pool, v_pool = (torch.randn(shape, device=DEV, generator=g).to(dtype) for _ in range(2))
    return dict(op="write", k=k, v=v, k_pool=k_pool, v_pool=v_pool, slots=slots, rows=rows, pages=pages)


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    s = state
    if own:
        return _own(s)
    return {"attention": _plain_attention, "masks": _plain_masks, "accept": _plain_accept, "tables": _plain_tables, "write": _plain_write}[s["op"]](s)


def _own(s):
    from actfold_b200 import speculative as spec

    if s["op"] == "attention":
        return {"out": spec.tree_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lengths"], s["starts"], s["mask"])}
    if s["op"] == "masks":
        mask, positions = spec.tree_masks(s["parents"], s["starts"], s["words"], s["base"])
        return {"mask": mask, "positions": positions}
    if s["op"] == "accept":
        r = spec.accept_tree(s["parents"], s["tokens"], s["targets"], s["starts"], s["keep"], s["root_targets"])
        return {"rows": r.rows, "counts": r.counts, "next_tokens": r.next_tokens}
    if s["op"] == "tables":
        r = spec.block_tables(s["tables"], s["lengths"], s["grow"], s["free"], s["free_range"], s["page"], s["capacity"], held=s["held"])
        return {"tables": s["tables"], "free": s["free"], "starts": r.starts, "totals": r.totals, "slots": r.slots, "free_range": r.free_range}
    k_cache, v_cache = s["k_pool"][:, : s["pages"]], s["v_pool"][:, : s["pages"]]
    spec.write_cache(s["k"], s["v"], k_cache, v_cache, s["slots"], rows=s["rows"])
    return {"k_cache": k_cache, "v_cache": v_cache}


def _plain_attention(s):
    """Every request padded to the longest: out = softmax(q k^T / sqrt(dim)) v over the cached keys and the tree's visible ones."""
    q, starts, lengths, tables = s["q"], s["starts"].long(), s["lengths"].long(), s["tables"].long()
    total, heads, dim = q.shape
    page, kv = s["k_cache"].shape[1:3]
    n, t, b = s["most_nodes"], s["longest"], tables.shape[0]
    node = torch.arange(n, device=DEV)
    there = node < (starts[1:] - starts[:-1])[:, None]  # [b, n]
    row = (starts[:-1, None] + node).clamp(max=total - 1)
    position = torch.arange(t, device=DEV)
    slot = tables[:, position // page].clamp(min=0) * page + position % page  # [b, t]
    k = torch.cat([s["k_cache"].reshape(-1, kv, dim)[slot], s["k"][row]], 1).float()  # [b, t + n, kv, dim]
    v = torch.cat([s["v_cache"].reshape(-1, kv, dim)[slot], s["v"][row]], 1).float()
    if s["mask"] is None:
        sees = (node <= node[:, None]).expand(b, n, n)
    else:
        sees = ((s["mask"][row][..., node // 32] >> (node % 32)) & 1).bool()  # [b, n, n]
    sees = torch.cat([(position < lengths[:, None])[:, None].expand(b, n, t), sees & there[:, None]], 2)
    x = q[row].float().view(b, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)  # rows: head of the group, node
    scores = (x @ k.permute(0, 2, 3, 1) * dim ** -0.5).view(b, kv, heads // kv, n, t + n)
    scores = torch.where(sees[:, None, None], scores, -math.inf)
    del k
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total_p = scores.sum(-1, keepdim=True)
    out = scores.view(b, kv, -1, t + n) @ v.permute(0, 2, 1, 3)
    out = out.view(b, kv, -1, n, dim) / torch.where(total_p > 0, total_p, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(b * n, heads, dim)
    place = torch.repeat_interleave(torch.arange(b, device=DEV) * n - starts[:-1], starts[1:] - starts[:-1], output_size=total)
    return {"out": out[place + torch.arange(total, device=DEV)].to(q.dtype)}


def _closure(parents, starts, words):
    """(which request a node is of, ancestor matrix over its own tree, its row of the parent or the sentinel row, depth), by doubling the step to the root."""
    total = parents.numel()
    of = torch.searchsorted(starts[1:].contiguous(), torch.arange(total, device=DEV, dtype=starts.dtype), right=True)
    first = starts.long()[of]
    jump = torch.cat([torch.where(parents < 0, total, parents.long() + first), _ints([total], torch.int64)])
    up = jump
    seen = torch.zeros(total + 1, 32 * words, dtype=torch.bool, device=DEV)
    seen[:total].scatter_(1, (torch.arange(total, device=DEV) - first)[:, None], True)
    depth = (jump != total).long()
    for _ in range(max(1, (32 * words - 1).bit_length())):
        seen, depth, jump = seen | seen[jump], depth + depth[jump], jump[jump]
    return of, seen[:total], up, depth[:total]


def _plain_masks(s):
    of, seen, _, depth = _closure(s["parents"], s["starts"], s["words"])
    bits = (seen.view(-1, s["words"], 32).long() << torch.arange(32, device=DEV)).sum(-1)
    return {"mask": torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32), "positions": (s["base"].long()[of] + depth).to(torch.int32)}


def _plain_accept(s):
    """A node is accepted when it and all its ancestors hold the token that the target model chose after their parents; the deepest one ends the path
    (of several, the first), which is cut to `keep` nodes."""
    starts, keep, b = s["starts"].long(), s["keep"], s["batch"]
    of, seen, up, depth = _closure(s["parents"], s["starts"], s["words"])
    total = of.numel()
    wanted = torch.where(up[:total] == total, s["root_targets"][of], s["targets"][up[:total].clamp(max=total - 1)])
    wrong = s["tokens"] != wanted
    local = torch.arange(total, device=DEV) - starts[of]
    square = torch.zeros(b, seen.shape[1], dtype=torch.bool, device=DEV)
    square[of, local] = wrong
    good = ~(seen & square[of]).any(1)
    key = torch.where(good, (depth + 1) * 65536 + 65535 - local, 0)
    best = torch.zeros(b, dtype=torch.int64, device=DEV).scatter_reduce(0, of, key, "amax")
    some = best > 0
    end = starts[:-1] + 65535 - best % 65536
    path = seen[end.clamp(max=total - 1)] & some[:, None]
    rank = path.long().cumsum(1) - 1
    path = path & (rank < keep)
    rows = torch.full((b, keep + 1), -1, dtype=torch.int64, device=DEV)
    rows.scatter_(1, torch.where(path, rank, keep), torch.where(path, starts[:-1, None] + torch.arange(seen.shape[1], device=DEV), -1))
    rows = rows[:, :keep]
    counts = (rows >= 0).sum(1)
    last = rows.gather(1, (counts - 1).clamp(min=0)[:, None])[:, 0]
    following = torch.where(counts > 0, s["targets"][last.clamp(min=0)], s["root_targets"])
    return {"rows": rows.to(torch.int32), "counts": counts.to(torch.int32), "next_tokens": following}


def _plain_tables(s):
    """Pages that a request no longer needs go to the end of the ring of free pages, pages that it lacks come from its front, both in the order of requests."""
    page, free = s["page"], s["free"].long()
    tables, (b, most) = s["tables"].long(), s["tables"].shape
    pool, head, tail = free.numel(), s["free_range"][0], s["free_range"][1]
    totals = (s["lengths"] + s["grow"]).long()
    had, wants = (s["held"].long() + page - 1) // page, (totals + page - 1) // page
    more, less = (wants - had).clamp(min=0), (had - wants).clamp(min=0)
    entry = torch.arange(most, device=DEV)
    taken = (entry >= had[:, None]) & (entry < wants[:, None])
    source = (head + (more.cumsum(0) - more)[:, None] + entry - had[:, None]) % pool
    left = (entry >= wants[:, None]) & (entry < had[:, None])
    target = torch.where(left, (tail + (less.cumsum(0) - less)[:, None] + entry - wants[:, None]) % pool, pool)
    ring = torch.cat([free, free[:1]])
    ring[target] = tables
    tables = torch.where(taken, free[source], tables)
    starts = torch.cat([_zero(), s["grow"].long().cumsum(0)])
    token = torch.arange(s["capacity"], device=DEV)
    of = torch.searchsorted(starts[1:].contiguous(), token, right=True).clamp(max=b - 1)
    position = s["lengths"].long()[of] + token - starts[of]
    slots = tables[of, (position // page).clamp(max=most - 1)] * page + position % page
    slots = torch.where(token < starts[-1], slots, -1)
    return {"tables": tables.to(torch.int32), "free": ring[:pool].to(torch.int32), "starts": starts.to(torch.int32), "totals": totals.to(torch.int32),
            "slots": slots, "free_range": torch.stack([head + more.sum(), tail + less.sum()])}


def _zero():
    return torch.zeros(1, dtype=torch.int64, device=DEV)


def _plain_write(s):
    layers, _, page, heads, dim = s["k_pool"].shape
    slots = s["slots"].reshape(-1)
    slots = torch.where(slots < 0, s["pages"] * page, slots)  # to the page that nobody is given
    k, v = s["k"], s["v"]
    if s["rows"] is not None:
        rows = s["rows"].reshape(-1).clamp(min=0)
        k, v = k[:, rows], v[:, rows]
    s["k_pool"].view(layers, -1, heads, dim)[:, slots] = k
    s["v_pool"].view(layers, -1, heads, dim)[:, slots] = v
    return {"k_cache": s["k_pool"][:, : s["pages"]], "v_cache": s["v_pool"][:, : s["pages"]]}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Request by request in 64 bits. The operators on whole numbers have nothing to be off by."""
    if case["op"] not in ("attention", "write"):
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        kc, vc = s["k_pool"][:, : s["pages"]].double(), s["v_pool"][:, : s["pages"]].double()
        page = kc.shape[2]
        slots = s["slots"].reshape(-1).tolist()
        rows = list(range(len(slots))) if s["rows"] is None else s["rows"].reshape(-1).tolist()
        for r, x in zip(rows, slots):
            if x >= 0:
                kc[:, x // page, x % page] = s["k"][:, r].double()
                vc[:, x // page, x % page] = s["v"][:, r].double()
        return {"k_cache": kc, "v_cache": vc}
    group, dim = case["heads"] // case["kv_heads"], case["dim"]
    edges, lengths = s["starts"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, t in enumerate(lengths):
        lo, hi = edges[r], edges[r + 1]
        pages = s["tables"][r, : _pages(t, case["page"])].long()
        k, v = (torch.cat([x[pages].flatten(0, 1)[:t], y[lo:hi]]) for x, y in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])))
        count = hi - lo
        hidden = torch.zeros(count, t + count, dtype=torch.bool, device=DEV)
        if s["mask"] is None:
            hidden[:, t:] = torch.ones(count, count, dtype=torch.bool, device=DEV).triu(1)
        else:
            words = s["mask"][lo:hi].long() & 0xFFFFFFFF
            hidden[:, t:] = torch.stack([(words[:, j // 32] >> (j % 32)) & 1 for j in range(count)], 1) == 0
        for h in range(case["heads"]):
            scores = s["q"][lo:hi, h].double() @ k[:, h // group].double().T / math.sqrt(dim)
            out[lo:hi, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v[:, h // group].double()
    return {"out": out}
