"""Tree verification operators against plain 64-bit forms.

Whole numbers (tables, slots, masks, paths) and copied rows must be equal. The
attention's tolerance is derived in tree_util.attention: the rounding of the
probabilities and of the result to the inputs' type (half a step each) plus
the 32-bit arithmetic's, element by element.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tree_util as U

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(ns):
    return [0, *np.cumsum(ns).tolist()]


# ------------------------------------------------------------------------------------------------ masks
@pytest.mark.parametrize("ns,words", [([1], 1), ([26], 1), ([0, 5, 0, 33, 64, 1], 2), ([128, 129, 127], 5), ([700, 3], 22), ([0, 0], 1)])
def test_masks_and_positions(ns, words):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_masks

    rng = np.random.default_rng(sum(ns) + words)
    trees = [U.random_parents(n, rng) for n in ns]
    base = [int(x) for x in rng.integers(0, 100000, len(ns))]
    st = DeviceStatus()
    mask, pos = tree_masks(_i32([p for t in trees for p in t]), _i32(_starts(ns)), words, _i32(base), status=st)
    st.check_status()
    paths = [U.ancestors(t) for t in trees]
    want = np.concatenate([U.pack_bits(p, words) for p in paths]) if sum(ns) else np.zeros((0, words), np.int32)
    assert np.array_equal(mask.cpu().numpy(), want)
    assert pos.tolist() == [b + len(x) - 1 for b, p in zip(base, paths) for x in p]


def test_masks_of_a_deep_chain_and_without_base():
    from actfold_b200.speculative import tree_masks

    n = 1000
    mask, pos = tree_masks(_i32(list(range(-1, n - 1))), _i32([0, n]), 32)
    assert pos.tolist() == list(range(n))
    assert np.array_equal(mask.cpu().numpy(), U.pack_bits([list(range(i + 1)) for i in range(n)], 32))


def test_masks_report_bad_trees_and_do_the_others():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_masks

    st = DeviceStatus()
    # Tree 0: node 1's parent is itself; tree 1 is longer than 32 nodes; tree 2 is sound.
    parents = [-1, 1, 0] + [-1] * 40 + [-1, 0, 1]
    mask, pos = tree_masks(_i32(parents), _i32([0, 3, 43, 46]), 1, status=st)
    with pytest.raises(RuntimeError):
        st.check_status()
    assert mask[43:, 0].tolist() == [1, 3, 7] and pos[43:].tolist() == [0, 1, 2]
    st2 = DeviceStatus()
    tree_masks(_i32([-1, 0]), _i32([0, 5]), 1, status=st2)  # starts behind the last node
    with pytest.raises(RuntimeError):
        st2.check_status()


def test_masks_with_torchs_public_names_of_device_and_stream(monkeypatch):
    from actfold_b200 import _lib
    from actfold_b200 import tree_kernels as T

    monkeypatch.setattr(T, "_current_device", torch.cuda.current_device)
    monkeypatch.setattr(T, "_current_stream", _lib.stream_ptr)
    parents, starts = _i32([-1, 0, 1]), _i32([0, 3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        mask, _ = T.tree_masks(parents, starts, 1)
    s.synchronize()
    assert mask[:, 0].tolist() == [1, 3, 7]


@pytest.mark.parametrize("ns,words", [([1200, 5, 1100], 38), ([1025, 0, 2000, 1], 64), ([31, 1056, 32], 33)])
def test_masks_of_branching_trees_with_more_than_32_words(ns, words):
    """Rows that go straight out: every word of every row, the zero ones among them, of several trees."""
    test_masks_and_positions(ns, words)


# ------------------------------------------------------------------------------------------------ acceptance
@pytest.mark.parametrize("ns,keep,vocab,with_root", [([26], 6, 3, True), ([1, 0, 7, 300], 4, 2, True), ([40, 41], 64, 1, True),
                                                     ([300, 5], 300, 1, False), ([9, 0, 12], 1, 2, False), ([600], 8, 5, True)])
def test_accept(ns, keep, vocab, with_root):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import accept_tree

    rng = np.random.default_rng(keep + sum(ns))
    trees = [U.random_parents(n, rng, chain=0.6) for n in ns]
    total = sum(ns)
    tokens, targets = (rng.integers(0, vocab, total) + 2 ** 40 for _ in range(2))
    root = rng.integers(0, vocab, len(ns)) + 2 ** 40
    starts = _starts(ns)
    st = DeviceStatus()
    got = accept_tree(_i32([p for t in trees for p in t]), torch.from_numpy(tokens).cuda(), torch.from_numpy(targets).cuda(), _i32(starts), keep,
                      torch.from_numpy(root).cuda() if with_root else None, status=st)
    st.check_status()
    for b, t in enumerate(trees):
        lo, hi = starts[b], starts[b + 1]
        path, nxt = U.accept(t, tokens[lo:hi].tolist(), targets[lo:hi].tolist(), int(root[b]) if with_root else None, keep)
        assert got.rows[b].tolist() == [lo + x for x in path] + [-1] * (keep - len(path))
        assert got.counts[b].item() == len(path) and got.next_tokens[b].item() == nxt


def test_accept_ties_and_bad_parents():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import accept_tree

    tok = torch.full((4,), 5, dtype=torch.int64, device="cuda")
    st = DeviceStatus()
    # Two paths of length two with equal tokens: the first one; node 3 is its own parent and is left out.
    got = accept_tree(_i32([-1, 0, 0, 3]), tok, tok, _i32([0, 4]), 3, torch.full((1,), 5, dtype=torch.int64, device="cuda"), status=st)
    assert got.rows.tolist() == [[0, 1, -1]] and got.counts.tolist() == [2]
    with pytest.raises(RuntimeError):
        st.check_status()
    got = accept_tree(_i32([-1, 0, 0, 3]), tok, tok, _i32([0, 4]), 3, max_nodes=3, status=st)  # a tree larger than was said
    assert got.counts.tolist() == [0] and got.next_tokens.tolist() == [-1]
    with pytest.raises(RuntimeError):
        st.check_status()


def test_accept_from_a_branch_tree():
    from actfold_b200 import speculative as S

    tree = S.BranchTree(S.BranchNode("root", None, torch.tensor([[5, 6]], device="cuda")))
    texts = {"a": [7], "b": [8], "aa": [7, 1], "ba": [8, 2], "bb": [8, 3], "baa": [8, 2, 4]}
    for name, t in texts.items():
        tree.add(S.BranchNode(name, name[:-1] or "root", torch.tensor([[5, 6, *t]], device="cuda")))
    ids, parents, tokens = tree.packed()
    starts = _i32([0, len(ids)])
    choice = {"root": 8, "a": 1, "b": 2, "aa": 0, "ba": 9, "bb": 0, "baa": 0}  # what the target model would say after each
    targets = torch.tensor([choice[i] for i in ids], device="cuda")
    got = S.accept_tree(parents, tokens, targets, starts, 4, torch.tensor([8], device="cuda"))
    kept = [ids[i] for i in got.rows[0].tolist() if i >= 0]
    assert kept == ["b", "ba"] and got.next_tokens.tolist() == [9]
    mask, _ = S.tree_masks(parents, starts, 1)
    for i, name in enumerate(ids):
        assert mask[i, 0].item() == sum(1 << ids.index(name[: k + 1]) for k in range(len(name)))


# ------------------------------------------------------------------------------------------------ block tables
def _pool(batch, most, held, page, spare, rng, head):
    used = [-(-h // page) for h in held]
    pool = sum(used) + spare
    order = rng.permutation(pool).tolist()
    tables = [[-1] * most for _ in range(batch)]
    at = 0
    for r, u in enumerate(used):
        tables[r][:u] = order[at: at + u]
        at += u
    ring = [-7] * pool
    for i, x in enumerate(order[at:]):
        ring[(head + i) % pool] = x
    return tables, ring, head, head + spare


@pytest.mark.parametrize("batch,page,top,grow_to,padded", [(1, 16, 40, 5, 0), (5, 16, 100, 9, 0), (7, 1, 9, 4, 5), (33, 100, 700, 400, 0),
                                                           (1500, 8, 60, 6, 8), (3, 64, 3000, 9000, 0)])
def test_block_tables(batch, page, top, grow_to, padded):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import block_tables

    rng = np.random.default_rng(batch * 7 + page)
    held = rng.integers(0, top + 1, batch)
    held[rng.random(batch) < 0.2] = 0
    kept = np.maximum(0, held - rng.integers(0, 2 * page + 2, batch))
    kept[rng.random(batch) < 0.2] = 0
    grow = rng.integers(0, (min(padded, grow_to) if padded else grow_to) + 1, batch)
    most = max(-(-max(h, k + g) // page) for h, k, g in zip(held, kept, grow)) + 1
    need = sum(max(0, -(-(k + g) // page) - -(-h // page)) for h, k, g in zip(held, kept, grow))
    tables, ring, head, tail = _pool(batch, most, held.tolist(), page, int(need) + 2, rng, 1000 + batch)
    want = U.tables_step(tables, held.tolist(), kept.tolist(), grow.tolist(), ring, head, tail, page)
    tt, rr = _i32(tables), _i32(ring)
    st = DeviceStatus()
    cap = padded or int(grow.sum()) + 3
    got = block_tables(tt, _i32(kept.tolist()), _i32(grow.tolist()), rr, torch.tensor([head, tail], device="cuda"), page, cap,
                       held=_i32(held.tolist()), padded=bool(padded), status=st)
    st.check_status()
    assert tt.tolist() == want[0] and rr.tolist() == want[1]
    assert got.free_range.tolist() == [want[3], want[4]]
    assert got.starts.tolist() == _starts(grow.tolist()) and got.totals.tolist() == (kept + grow).tolist()
    if padded:
        assert got.slots.tolist() == [s + [-1] * (padded - len(s)) for s in want[2]]
    else:
        assert got.slots.tolist() == [x for s in want[2] for x in s] + [-1] * 3


@pytest.mark.parametrize("why", ["pages", "row", "slots", "negative", "ring", "padded"])
def test_block_tables_that_do_not_fit_change_nothing(why):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import block_tables

    rng = np.random.default_rng(3)
    held, kept, grow, cap, page = [20, 0, 33], [18, 0, 30], [9, 25, 4], 50, 8
    tables, ring, head, tail = _pool(3, 6, held, page, 4 if why == "pages" else 20, rng, 5)
    if why == "row":
        grow[0] = 40
    if why == "slots":
        cap = 30
    if why == "negative":
        kept[1] = -1
    if why == "ring":
        tail = head - 1
    if why == "padded":
        cap = 24
    tt, rr, st = _i32(tables), _i32(ring), DeviceStatus()
    got = block_tables(tt, _i32(kept), _i32(grow), rr, torch.tensor([head, tail], device="cuda"), page, cap, held=_i32(held),
                       padded=why == "padded", status=st)
    assert tt.tolist() == tables and rr.tolist() == ring and got.free_range.tolist() == [head, tail]
    assert got.starts.tolist() == [0] * 4 and got.totals.tolist() == held and set(got.slots.flatten().tolist()) == {-1}
    with pytest.raises(RuntimeError):
        st.check_status()


@pytest.mark.parametrize("where", ["taken", "returned", "last returned"])
@pytest.mark.parametrize("batch", [3, 1500])
def test_block_tables_with_an_entry_that_is_no_page_change_nothing(where, batch):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import block_tables

    rng = np.random.default_rng(5)
    page = 8
    held = [20, 0, 33] * (batch // 3)
    kept, grow = [18, 0, 3] * (batch // 3), [9, 25, 2] * (batch // 3)  # of three requests one grows, one is new, one gives pages back
    tables, ring, head, tail = _pool(batch, 6, held, page, 5 * batch, rng, 7)
    pool = len(ring)
    if where == "taken":
        ring[(head + 2 * batch // 3) % pool] = -1
    elif where == "returned":
        tables[2][3] = -3
    else:
        tables[batch - 1][4] = -1
    tt, rr, st = _i32(tables), _i32(ring), DeviceStatus()
    got = block_tables(tt, _i32(kept), _i32(grow), rr, torch.tensor([head, tail], device="cuda"), page, sum(grow), held=_i32(held), status=st)
    assert tt.tolist() == tables and rr.tolist() == ring and got.free_range.tolist() == [head, tail]
    assert set(got.starts.tolist()) == {0} and got.totals.tolist() == held and set(got.slots.tolist()) == {-1}
    with pytest.raises(RuntimeError):
        st.check_status()


def test_block_tables_report_a_held_entry_that_is_no_page():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import block_tables

    # The page that request 0 goes on in is missing; request 1 is sound.
    tables, ring, st = _i32([[4, -1, -1], [2, -1, -1]]), _i32([5, 6, 7]), DeviceStatus()
    got = block_tables(tables, _i32([12, 6]), _i32([6, 3]), ring, torch.tensor([0, 3], device="cuda"), 8, 9, status=st)
    assert got.slots.tolist() == [-1] * 4 + [40, 41, 22, 23, 48] and got.totals.tolist() == [18, 9]
    assert tables.tolist() == [[4, -1, 5], [2, 6, -1]] and got.free_range.tolist() == [2, 3]
    with pytest.raises(RuntimeError):
        st.check_status()
    # An entry in front of the kept tokens' last page is not looked at.
    tables = _i32([[-1, 3]])
    assert block_tables(tables, _i32([9]), _i32([2]), ring, torch.tensor([0, 3], device="cuda"), 8, 2, status=st).slots.tolist() == [25, 26]
    st.check_status()


def test_block_tables_over_many_steps_keep_every_page_once():
    from actfold_b200.speculative import block_tables

    rng = np.random.default_rng(11)
    batch, page, most, pool = 9, 16, 12, 90
    tables, ring = torch.full((batch, most), -1, dtype=torch.int32, device="cuda"), _i32(rng.permutation(pool).tolist())
    span = torch.tensor([0, pool], device="cuda")
    plain = ([[-1] * most for _ in range(batch)], ring.tolist(), None, 0, pool)
    held = [0] * batch
    for step in range(40):
        kept = [int(rng.integers(max(0, h - 20), h + 1)) if rng.random() > 0.1 else 0 for h in held]
        grow = [int(rng.integers(0, min(30, most * page - k) + 1)) for k in kept]
        plain = U.tables_step(plain[0], held, kept, grow, plain[1], plain[3], plain[4], page)
        got = block_tables(tables, _i32(kept), _i32(grow), ring, span, page, 300, held=_i32(held))
        span, held = got.free_range, [k + g for k, g in zip(kept, grow)]
        owned = [x for r, h in zip(tables.tolist(), held) for x in r[: -(-h // page)]]
        head, tail = span.tolist()
        free = [ring.tolist()[e % pool] for e in range(head, tail)]
        assert sorted(owned + free) == list(range(pool))
        assert tables.tolist() == plain[0] and [head, tail] == list(plain[3:])


@pytest.mark.parametrize("batch", [4031, 4032, 4095, 4096])
def test_block_tables_where_the_sums_pass_the_default_shared_memory(batch):
    """Three sums per request and the static state: 48 KB lie between 4031 and 4096 requests."""
    from actfold_b200.speculative import block_tables

    tables = torch.full((batch, 2), -1, dtype=torch.int32, device="cuda")
    kept, grow = [0] * batch, [r % 3 for r in range(batch)]
    ring, span = _i32(list(range(batch))), torch.tensor([0, batch], device="cuda")
    want = U.tables_step(tables.tolist(), kept, kept, grow, ring.tolist(), 0, batch, 16)
    got = block_tables(tables, _i32(kept), _i32(grow), ring, span, 16, sum(grow))
    assert tables.tolist() == want[0] and got.slots.tolist() == [x for r in want[2] for x in r]
    assert got.free_range.tolist() == list(want[3:])


@pytest.mark.parametrize("n", [12270, 12288, 12320])
def test_trees_whose_parents_pass_the_default_shared_memory(n):
    """A chain per tree; 48 KB of parents are 12288 nodes."""
    from actfold_b200.speculative import accept_tree, tree_masks

    parents, starts = _i32(list(range(-1, n - 1))), _i32([0, n])
    words = -(-n // 32)
    mask, positions = tree_masks(parents, starts, words)
    assert positions.tolist() == list(range(n))
    last = [-1] * (n // 32) + ([(1 << n % 32) - 1] if n % 32 else [])
    assert mask[-1].tolist() == last
    tokens = torch.arange(n, device="cuda")
    path = accept_tree(parents, tokens, tokens + 1, starts, 5, root_targets=torch.tensor([0], device="cuda"))
    assert path.rows.tolist() == [[0, 1, 2, 3, 4]] and path.counts.tolist() == [5] and path.next_tokens.tolist() == [5]


# ------------------------------------------------------------------------------------------------ cache writes
@pytest.mark.parametrize("layers,heads,dim,dtype,page", [(1, 32, 128, torch.bfloat16, 64), (3, 4, 128, torch.float16, 16), (2, 1, 64, torch.float32, 5),
                                                         (1, 3, 5, torch.bfloat16, 7), (2, 5, 6, torch.int8, 16), (1, 2, 80, torch.float16, 48)])
@pytest.mark.parametrize("gathered", [False, True])
def test_write_cache(layers, heads, dim, dtype, page, gathered):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import write_cache

    g = torch.Generator(device="cuda").manual_seed(heads + dim)
    n, pages = 37, 11

    def rand(*shape):
        return (torch.randn(*shape, device="cuda", generator=g) * 40).to(dtype)

    k, v = rand(layers, n, heads, dim), rand(layers, n, heads, dim)
    kc, vc = rand(layers, pages, page, heads, dim), rand(layers, pages, page, heads, dim)
    m = 24 if gathered else n
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:m].clone()
    slots[3] = -1
    rows = torch.randint(0, n, (m,), device="cuda", generator=g, dtype=torch.int32) if gathered else None
    if gathered:
        rows[5] = -1
        slots, rows = slots.view(4, 6), rows.view(4, 6)
    wk, wv = kc.clone(), vc.clone()
    for i, s in enumerate(slots.flatten().tolist()):
        r = rows.flatten()[i].item() if gathered else i
        if s >= 0 and r >= 0:
            wk[:, s // page, s % page], wv[:, s // page, s % page] = k[:, r], v[:, r]
    st = DeviceStatus()
    write_cache(k, v, kc, vc, slots, rows=rows, status=st)
    st.check_status()
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_write_cache_strided_transposed_and_single_layer():
    from actfold_b200.speculative import write_cache

    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(19, 12, 128, device="cuda", generator=g).to(torch.bfloat16)  # 4 query, 4 key, 4 value heads
    cache = torch.zeros(2, 6, 4, 16, 128, dtype=torch.bfloat16, device="cuda")  # [k / v, page, head, token, dim]
    slots = torch.randperm(96, device="cuda", generator=g)[:19]
    write_cache(qkv[:, 4:8], qkv[:, 8:], cache[0].transpose(1, 2), cache[1].transpose(1, 2), slots)
    want = torch.zeros_like(cache)
    for i, s in enumerate(slots.tolist()):
        want[0, s // 16, :, s % 16], want[1, s // 16, :, s % 16] = qkv[i, 4:8], qkv[i, 8:]
    assert torch.equal(cache, want)
    off = torch.zeros(6 * 16 * 4 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 16, 4, 128)  # off the 16-byte grid
    write_cache(qkv[:, 4:8], qkv[:, 8:], off, torch.zeros_like(off), slots)
    assert torch.equal(off.transpose(1, 2), want[0])


def test_write_cache_skips_slots_and_rows_out_of_range():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import write_cache

    k = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    cache = torch.zeros(4, 8, 2, 64, dtype=torch.float16, device="cuda")
    st = DeviceStatus()
    write_cache(k, k, cache, cache.clone(), torch.tensor([32, 5, 9], device="cuda"), rows=_i32([0, 3, 1]), status=st)
    with pytest.raises(RuntimeError):
        st.check_status()
    assert cache[1, 1].eq(1).all() and cache.sum().item() == 128


@pytest.mark.parametrize("none", ["rows", "pages"])
def test_write_cache_of_a_step_without_rows_or_pages(none):
    """No node in any tree, or a pool without pages: every entry is skipped, and one that is not negative is reported."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import write_cache

    k = torch.ones(2, 0 if none == "rows" else 4, 2, 64, dtype=torch.float16, device="cuda")
    cache = torch.zeros(2, 0 if none == "pages" else 3, 8, 2, 64, dtype=torch.float16, device="cuda")
    slots, rows, st = torch.full((3, 5), -1, device="cuda"), torch.full((3, 5), -1, dtype=torch.int32, device="cuda"), DeviceStatus()
    write_cache(k, k, cache, cache.clone(), slots, rows=rows, status=st)
    st.check_status()
    write_cache(k, k, cache, cache.clone(), torch.full_like(slots, 3), rows=rows, status=st)
    st.check_status()
    rows[1, 2], slots[1, 2] = 1, 3
    write_cache(k, k, cache, cache.clone(), slots, rows=rows, status=st)
    with pytest.raises(RuntimeError):
        st.check_status()
    assert not cache.any()


def test_write_cache_far_offsets():
    """A cache of more than 2^32 bytes: its last slots."""
    from actfold_b200.speculative import write_cache

    k = torch.randn(2, 8, 128, device="cuda").to(torch.bfloat16)
    cache = torch.zeros(20000, 64, 8, 128, dtype=torch.bfloat16, device="cuda")  # 2.6 GB: 2^31 bytes are passed
    vcache = torch.zeros(40000, 64, 8, 128, dtype=torch.bfloat16, device="cuda")[::2]  # strided pages: 2^32 bytes are passed
    slots = torch.tensor([20000 * 64 - 1, 17000 * 64 + 3], device="cuda")
    write_cache(k, k, cache, vcache, slots)
    for c in (cache, vcache):
        assert torch.equal(c[19999, 63], k[0]) and torch.equal(c[17000, 3], k[1])


# ------------------------------------------------------------------------------------------------ attention
def _case(lengths, ns, heads, kv, dim, page, dtype, seed=0, kind="tree", hnd=False, spread=1.0, extra=0):
    """Inputs with NaN in every place that no row may see: spare pages, page ends, rows behind the last tree."""
    rng = np.random.default_rng(seed + 1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-t // page) for t in lengths]
    pages = sum(used) + 2
    order = rng.permutation(pages).tolist()
    most = max(1, max(used, default=0))
    tables, at = [], 0
    for u in used:
        tables.append(order[at: at + u] + [-1] * (most - u))
        at += u
    total = sum(ns)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    q = (rand(total + extra, heads, dim) * spread).to(dtype)
    k, v = rand(total + extra, kv, dim).to(dtype), rand(total + extra, kv, dim).to(dtype)
    shape = (pages, kv, page, dim) if hnd else (pages, page, kv, dim)
    kc, vc = rand(*shape).to(dtype), rand(*shape).to(dtype)
    if hnd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    for b, t in enumerate(lengths):
        if t % page:
            kc[tables[b][used[b] - 1], t % page:] = float("nan")
            vc[tables[b][used[b] - 1], t % page:] = float("nan")
    for x in order[at:]:
        kc[x], vc[x] = float("nan"), float("inf")
    k[total:], v[total:], q[total:] = float("nan"), float("nan"), float("nan")
    words = max(1, -(-max(ns, default=1) // 32))
    bits, rows = [], []
    for n in ns:
        if kind == "tree":
            see = U.ancestors(U.random_parents(n, rng))
        elif kind == "any":  # any bits, rows of nothing among them
            see = [[j for j in range(n) if rng.random() < 0.4] if rng.random() < 0.7 else [] for _ in range(n)]
        elif kind == "none":
            see = [[] for _ in range(n)]
        else:
            see = [list(range(i + 1)) for i in range(n)]
        m = torch.zeros(n, n, dtype=torch.bool)
        for i, r in enumerate(see):
            m[i, r] = True
        bits.append(m)
        rows += see
    mask = None if kind == "chain" else torch.from_numpy(U.pack_bits(rows + [[]] * extra, words)).cuda()
    return dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, tables=_i32(tables), lengths=_i32(lengths), starts=_i32(_starts(ns)), mask=mask), \
        (tables, lengths, _starts(ns), bits)


def _check(args, plain, scale=None, **kw):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    tables, lengths, starts, bits = plain
    st = DeviceStatus()
    lse = torch.full(args["q"].shape[:2], 7.0, device="cuda")
    out = tree_attention(**args, scale=scale, lse=lse, status=st, **kw)
    st.check_status()
    total = starts[-1]
    ref, ref_lse, tol, lse_tol = U.attention(args["q"], args["k"], args["v"], args["k_cache"], args["v_cache"], tables, lengths, starts, bits, scale)
    err = (out.double() - ref).abs()[:total]
    assert bool((err <= tol[:total]).all()), f"worst {float((err / tol[:total].clamp(min=1e-30)).max())} of the allowed error, max {float(err.max())}"
    got, want = lse[:total].double(), ref_lse[:total]
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fin = torch.isfinite(want)
    assert bool(((got - want).abs()[fin] <= lse_tol[:total][fin]).all())
    return out


CASES = [
    # lengths, nodes, heads, kv, dim, page, dtype, kind
    ([523], [1], 28, 4, 128, 16, torch.bfloat16, "chain"),
    ([0], [1], 2, 2, 128, 16, torch.bfloat16, "chain"),
    ([1], [1], 4, 1, 64, 8, torch.float16, "chain"),
    ([0, 0, 5], [3, 0, 1], 4, 2, 128, 16, torch.float16, "tree"),
    ([127, 128, 129, 255, 256, 257], [1, 2, 3, 1, 5, 1], 8, 2, 128, 32, torch.bfloat16, "tree"),
    ([100, 640, 33], [26, 64, 31], 8, 8, 128, 64, torch.bfloat16, "tree"),
    ([1000, 77], [64, 50], 28, 4, 128, 16, torch.float16, "tree"),
    ([300, 20], [130, 257], 4, 4, 128, 48, torch.bfloat16, "tree"),
    ([4000], [9], 16, 16, 64, 128, torch.bfloat16, "any"),
    ([200, 0, 64], [33, 40, 65], 6, 3, 64, 24, torch.float16, "any"),
    ([0, 0], [40, 12], 4, 4, 128, 16, torch.bfloat16, "none"),
    ([90], [6], 64, 1, 128, 104, torch.bfloat16, "tree"),
    ([700], [13], 33, 3, 128, 256, torch.float16, "tree"),
    ([50] * 70, [1] * 70, 28, 4, 128, 16, torch.bfloat16, "chain"),
    ([9000, 3, 2500], [1, 1, 1], 8, 2, 128, 64, torch.float16, "chain"),
    ([12, 2000], [300, 200], 2, 1, 128, 16, torch.bfloat16, "chain"),
    ([30000], [20], 4, 4, 128, 16, torch.bfloat16, "tree"),
    # more than 64 rows per key/value head: one row tile (even and odd key tiles), two, shared by several SMs or not
    ([7000], [100], 4, 4, 64, 32, torch.bfloat16, "any"),
    ([129, 4000, 0, 1], [70, 128, 90, 66], 4, 4, 128, 16, torch.bfloat16, "tree"),
    ([5000, 900], [64, 33], 28, 4, 128, 16, torch.float16, "tree"),
    ([6000, 40], [300, 5], 8, 2, 128, 64, torch.bfloat16, "any"),
    ([100, 1700], [129, 200], 6, 2, 64, 8, torch.float16, "chain"),
    ([0, 0, 3], [80, 200, 100], 2, 2, 128, 16, torch.bfloat16, "none"),
    ([20000], [64], 16, 1, 128, 48, torch.bfloat16, "tree"),
    # so long that every SM goes round its stages several times: 16, 32 and 64 rows per tile, and more
    ([150000], [2], 4, 2, 64, 32, torch.float16, "tree"),
    ([150000], [12], 4, 2, 64, 128, torch.bfloat16, "tree"),
    ([150000, 900], [25, 31], 4, 2, 64, 64, torch.float16, "tree"),
    ([150000], [90], 2, 2, 64, 32, torch.bfloat16, "tree"),
    ([100000], [2], 4, 2, 128, 32, torch.bfloat16, "tree"),
    ([100000, 100], [25, 31], 4, 2, 128, 64, torch.float16, "chain"),
]


@pytest.mark.parametrize("lengths,ns,heads,kv,dim,page,dtype,kind", CASES)
def test_attention(lengths, ns, heads, kv, dim, page, dtype, kind):
    args, plain = _case(lengths, ns, heads, kv, dim, page, dtype, seed=len(lengths) + sum(ns), kind=kind)
    _check(args, plain)


@pytest.mark.parametrize("case", [CASES[6], CASES[7], CASES[14], CASES[16], *CASES[17:]])
def test_attention_does_not_depend_on_what_its_scratch_held(case):
    """Rows that several SMs worked on are joined from scratch memory: only what this call wrote there may count."""
    from actfold_b200.speculative import tree_attention

    args, _ = _case(*case[:7], seed=2, kind=case[7])
    first = tree_attention(**args).clone()
    for i in range(6):
        junk = torch.full((12_000_000,), (float("nan"), 1e20, -3.0)[i % 3], device="cuda")  # freed at once: the next scratch lies in it
        del junk
        assert torch.equal(tree_attention(**args).view(torch.int16), first.view(torch.int16))


def test_attention_head_major_cache_and_fused_projections():
    args, plain = _case([333, 70], [9, 40], 8, 2, 128, 16, torch.bfloat16, hnd=True)
    fused = torch.cat([args["q"], args["k"], args["v"]], 1)
    args["q"], args["k"], args["v"] = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    _check(args, plain)


def test_attention_copies_rows_off_the_grid():
    args, plain = _case([40], [5], 4, 2, 64, 16, torch.float16)
    n = args["q"].numel()
    off = torch.empty(n + 1, dtype=torch.float16, device="cuda")[1:].view(args["q"].shape)
    off.copy_(args["q"])
    args["q"] = off
    args["k"] = args["k"].transpose(1, 2).contiguous().transpose(1, 2)
    _check(args, plain)


@pytest.mark.parametrize("spread,scale", [(8.0, None), (1.0, 1.0), (0.01, None), (30.0, None), (1.0, -0.2), (1.0, 0.0)])
@pytest.mark.parametrize("ns", [[3, 5], [20, 70]])
def test_attention_sharp_and_flat_rows(spread, scale, ns):
    args, plain = _case([1500, 200], ns, 8, 2, 128, 64, torch.bfloat16, spread=spread)
    _check(args, plain, scale=scale)


@pytest.mark.parametrize("step", [+1, -1])
@pytest.mark.parametrize("nodes", [7, 40, 80, 150])
def test_attention_maximum_that_moves_from_key_to_key(step, nodes):
    """Scores that rise (the running maximum is raised again and again) or fall along the cache."""
    args, plain = _case([2000], [nodes], 4, 4, 128, 16, torch.bfloat16)
    tables, (t,), _, _ = plain
    ramp = torch.linspace(0, 40, t, device="cuda") if step > 0 else torch.linspace(40, 0, t, device="cuda")
    args["q"][:, :, 0] = 11.3125  # about sqrt(128): the score gains the ramp
    for x in range(-(-t // 16)):
        part = ramp[16 * x: 16 * x + 16]
        args["k_cache"][tables[0][x], : len(part), :, 0] = part[:, None].to(torch.bfloat16)
    _check(args, plain)


@pytest.mark.parametrize("dim,nodes", [(128, 1), (64, 20), (128, 50), (128, 90), (64, 200)])
def test_attention_small_fp16_probabilities_count(dim, nodes):
    """In every 128 keys one that is far above the others, whose probabilities are 2^-24.9 to 2^-26 of its.

    The large keys' values are 0, the others' 1024, so the output is the sum of the small probabilities. Each is off by at most
    half a step of a subnormal fp16 number, 2^-25 of a largest one that the kernels hold at 2^7 or more: 1024 * 127 * 2^-32 in
    all; the result is rounded to fp16 (2^-11 relative), and the scores are off by 2^-24 (dim + 12) |s| in log2 terms.
    """
    from actfold_b200.speculative import tree_attention

    t, page = 4096, 64
    args, plain = _case([t], [nodes], 1, 1, dim, page, torch.float16, kind="none")
    order = torch.tensor(plain[0][0], device="cuda")
    keys, values = torch.zeros(t, dim, device="cuda"), torch.full((t, dim), 1024.0, device="cuda")
    keys[:, 0] = -torch.linspace(24.9, 26.0, t, device="cuda")
    keys[5::128], values[5::128] = 0.0, 0.0
    keys = keys.half()
    args["q"][:] = 0
    args["q"][:, :, 0] = 1
    args["k_cache"][order] = keys.view(-1, page, 1, dim)
    args["v_cache"][order] = values.half().view(-1, page, 1, dim)
    out = tree_attention(**args, scale=0.6931471805599453).double()  # scores in log2 are the keys' first entries
    e = torch.exp2(keys[:, 0].double())
    want = float((e * values[:, 0].double()).sum() / e.sum())
    allowed = 1024 * 127 * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -24 * (dim + 12) * 26)
    assert allowed < want / 50
    assert float((out - want).abs().max()) <= allowed


def test_attention_rows_behind_the_last_tree_stay():
    args, plain = _case([60, 5], [4, 30], 4, 2, 128, 16, torch.bfloat16, extra=6)
    out = torch.full_like(args["q"], 3.0)
    got = _check(args, plain, out=out)
    assert got is out and out[34:].eq(3.0).all()


@pytest.mark.parametrize("heads", [8, 2, 16])
def test_attention_hidden_nodes_have_no_influence(heads):
    """NaN and infinities in nodes (and in queries of others) that a row does not see."""
    args, plain = _case([200, 64, 0], [20, 3, 33], heads, 2, 128, 16, torch.bfloat16, kind="tree", seed=5)
    clean = _check(args, plain).clone()
    bits, starts = plain[3], plain[2]
    sick = [starts[0] + 19, starts[2] + 7]
    for s, x in zip(sick, (float("nan"), float("inf"))):
        args["k"][s], args["v"][s], args["q"][s] = float("nan"), x, x
    from actfold_b200.speculative import tree_attention

    out = tree_attention(**args)
    for b in range(3):
        for i in range(starts[b + 1] - starts[b]):
            if not any(starts[b] <= s < starts[b + 1] and bits[b][i, s - starts[b]] for s in sick):
                assert torch.equal(out[starts[b] + i], clean[starts[b] + i]), (b, i)
    assert out[sick[0]].isnan().all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads", [4, 32])
def test_attention_values_that_are_not_finite_reach_the_rows_that_see_them(value, heads):
    args, plain = _case([130], [12], heads, 2, 128, 16, torch.bfloat16, seed=8)
    args["v"][4, :, 3] = value
    from actfold_b200.speculative import tree_attention

    out = tree_attention(**args)
    sees = plain[3][0][:, 4].cuda()
    bad = ~torch.isfinite(out)
    assert torch.equal(bad[:, :, 3].all(1), sees) and not bad[:, :, :3].any() and not bad[:, :, 4:].any() and not bad[~sees].any()
    if value == value:
        assert (out[sees][:, :, 3] == value).all()


def test_attention_without_a_cache_or_without_nodes():
    from actfold_b200.speculative import tree_attention

    args, plain = _case([0, 0], [5, 40], 4, 2, 128, 16, torch.bfloat16)
    want = _check(args, plain)
    for pages in (0, 3):
        none = args["k_cache"][:0] if pages == 0 else args["k_cache"]
        got = tree_attention(**dict(args, k_cache=none, v_cache=none, tables=_i32([[], []]).view(2, 0)))
        assert torch.equal(got, want)
    e = args["q"][:0]
    assert tree_attention(**dict(args, q=e, k=args["k"][:0], v=args["v"][:0], mask=args["mask"][:0], starts=_i32([0, 0, 0]))).shape == e.shape
    out = torch.full_like(args["q"], 2.0)
    tree_attention(**dict(args, starts=_i32([0, 0, 0]), out=out))  # rows, but no tree
    assert out.eq(2.0).all()


def test_attention_reports_bad_pages_and_lengths():
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    args, plain = _case([40, 90, 16], [2, 3, 4], 4, 2, 128, 16, torch.bfloat16)
    good = _check(args, plain).clone()
    for key, at, value in (("tables", (1, 2), 10 ** 6), ("tables", (1, 2), -5), ("lengths", (1,), 10 ** 6), ("lengths", (1,), -3)):
        bad = dict(args)
        bad[key] = args[key].clone()
        bad[key][at] = value
        st = DeviceStatus()
        out = tree_attention(**bad, status=st)
        with pytest.raises(RuntimeError):
            st.check_status()
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[5:], good[5:]), (key, value)
    st = DeviceStatus()
    bad = dict(args, starts=_i32([0, 2, 1, 9]))
    tree_attention(**bad, status=st)
    with pytest.raises(RuntimeError):
        st.check_status()


@pytest.mark.parametrize("heads", [64, 2])
def test_attention_with_starts_out_of_order_writes_nothing(heads):
    """Trees that overlap 1500 times: more than 2^31 tiles with 64 key/value heads."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    n, batch, page = 3000, 3000, 64
    x = torch.ones(n, heads, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.ones(1, page, heads, 64, dtype=torch.bfloat16, device="cuda")
    starts = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = n
    tables, lengths = torch.zeros(batch, 256, dtype=torch.int32, device="cuda"), torch.full((batch,), 16384, dtype=torch.int32, device="cuda")
    out, st = torch.full_like(x, 5.0), DeviceStatus()
    tree_attention(x, x, x, cache, cache, tables, lengths, starts, out=out, status=st)
    with pytest.raises(RuntimeError):
        st.check_status()
    assert out.eq(5.0).all()


def test_attention_same_bits_again_and_on_another_stream():
    from actfold_b200.speculative import tree_attention

    args, _ = _case([3000, 800], [64, 20], 8, 4, 128, 16, torch.bfloat16)
    a = tree_attention(**args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = [tree_attention(**args) for _ in range(3)]
    c = tree_attention(**args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, x) for x in [*b, c])


def test_attention_far_offsets():
    """Pages beyond 2^32 bytes of a cache."""
    args, plain = _case([100], [3], 8, 8, 128, 64, torch.bfloat16)
    tables, lengths, starts, bits = plain
    big = torch.zeros(40000, 64, 8, 128, dtype=torch.bfloat16, device="cuda")[::2]
    far = [19999, 17777]
    kc, vc = big, big.clone()
    assert vc.is_contiguous()
    for x, y in zip(tables[0], far):
        kc[y], vc[y] = args["k_cache"][x], args["v_cache"][x]
    args.update(k_cache=kc, v_cache=vc, tables=_i32([far]))
    _check(args, ([far], lengths, starts, bits))


JOINED = [CASES[6], CASES[14], CASES[16], *CASES[17:20], *CASES[23:]]  # cases with rows that several SMs work on


@pytest.mark.parametrize("case", JOINED)
@pytest.mark.parametrize("junk", [0x7fc00000, 0x60ad78ec, -1, 0x3f800000])  # NaN, 1e20, all ones, 1
def test_attention_writes_all_of_its_scratch_that_it_reads(case, junk, monkeypatch):
    """The scratch memory is this test's own, filled with junk, and nothing behind its end is written."""
    from actfold_b200 import tree_kernels as T

    args, _ = _case(*case[:7], seed=2, kind=case[7])
    want = T.tree_attention(**args)
    size = T._workspace_bytes(0)
    scratch = torch.full((size // 4 + 64,), junk, dtype=torch.int32, device="cuda")
    launch, used = T._launch, []

    def with_own_scratch(what, index, fn, packed, *rest):
        fields = list(T._ATTENTION.unpack(packed))
        assert fields[-1] == size
        fields[-2] = scratch.data_ptr()
        used.append(what)
        launch(what, index, fn, T._ATTENTION.pack(*fields), *rest)

    monkeypatch.setattr(T, "_launch", with_own_scratch)
    got = T.tree_attention(**args)
    assert used == ["tree_attention"] and torch.equal(got, want)
    assert scratch[size // 4:].eq(junk).all() and not scratch[: size // 4].eq(junk).all()


@pytest.mark.parametrize("heads", [4, 64])  # narrow tiles and wide ones
def test_attention_with_a_mask_of_ones(heads):
    """Every bit of every word is set, those behind a tree's last node too: a node sees its own tree and nothing else."""
    ns = [33, 1, 7, 40]
    args, (tables, lengths, starts, _) = _case([100, 0, 300, 64], ns, heads, 2, 64, 16, torch.bfloat16)
    args["mask"] = torch.full((sum(ns), 3), -1, dtype=torch.int32, device="cuda")
    _check(args, (tables, lengths, starts, [torch.ones(n, n, dtype=torch.bool) for n in ns]))


def test_attention_of_the_most_requests():
    """16384 requests of one token (every seventh has none), a few keys each."""
    rng = np.random.default_rng(4)
    lengths, ns = rng.integers(0, 40, 16384).tolist(), [int(i % 7 > 0) for i in range(16384)]
    args, plain = _case(lengths, ns, 2, 1, 64, 8, torch.bfloat16, kind="chain")
    from actfold_b200.speculative import tree_attention

    out = tree_attention(**args)
    starts, some = plain[2], [0, 1, 2, 8, 5000, 11111, 16382, 16383]
    for b in some:
        if ns[b]:
            row = slice(starts[b], starts[b + 1])
            ref, _, tol, _ = U.attention(args["q"][row], args["k"][row], args["v"][row], args["k_cache"], args["v_cache"], [plain[0][b]], [lengths[b]],
                                         [0, 1], [None])
            assert bool(((out[row].double() - ref).abs() <= tol).all()), b
    assert out.isfinite().all()


def test_attention_of_many_requests_with_trees():
    rng = np.random.default_rng(9)
    lengths, ns = rng.integers(0, 700, 300).tolist(), rng.integers(0, 41, 300).tolist()
    _check(*_case(lengths, ns, 4, 2, 64, 16, torch.bfloat16))


def test_attention_on_two_streams_at_once_and_from_two_graphs():
    """Different inputs on each stream, calls in flight together; then the same from a graph each."""
    from actfold_b200.speculative import tree_attention

    cases = [_case([3000, 800], [64, 20], 8, 4, 128, 16, torch.bfloat16, seed=1)[0], _case([9000], [3], 8, 2, 128, 64, torch.float16, seed=2)[0],
             _case([2000, 77], [100, 90], 4, 4, 128, 32, torch.bfloat16, seed=3)[0]]
    want = [tree_attention(**a) for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, a, g in zip(streams, cases, got):
            with torch.cuda.stream(s):
                g.append(tree_attention(**a))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
    graphs, outs = [], []
    for a in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tree_attention(**a))
        graphs.append(graph)
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(w, x) for w, x in zip(want, outs))


@pytest.fixture
def wait_limit():
    """Sets how many attempts a wait inside the attention kernels makes; the default comes back at the end."""
    from actfold_b200 import _lib

    lib = _lib.load()
    yield lambda attempts: _lib.check(lib.af_tree_attention_wait_limit(attempts))
    torch.cuda.synchronize()
    _lib.check(lib.af_tree_attention_wait_limit(-1))


def _one_long_chain(n, heads, kv, dim, batch):
    """One chain of n nodes among empty requests, so that the average, which picks the kernel, is n / batch."""
    args, plain = _case([70], [n], heads, kv, dim, 16, torch.bfloat16, kind="none")
    args["mask"] = None
    more = batch - 1
    args["tables"] = torch.cat([args["tables"], torch.zeros(more, args["tables"].shape[1], dtype=torch.int32, device="cuda")])
    args["lengths"] = torch.cat([args["lengths"], _i32([0] * more)])
    args["starts"] = torch.cat([args["starts"], _i32([n] * more)])
    return args, plain


@pytest.mark.parametrize("group", [1, 4, 8, 16])  # tiles of 16, 32 and 64 rows, and the wide kernel
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_whose_waits_run_out_ends_with_a_status(group, dim, wait_limit):
    """Values that are not finite make the ends of rows long (their tiles are looked through for them): with a limit of one
    attempt the other warps' waits run out in the middle. The call ends and says so, and the next one is as always."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    n = 8000
    args, _ = _one_long_chain(n, 2 * group, 2, dim, n // 8)
    want = tree_attention(**args)
    sick = dict(args, v=args["v"].clone())
    sick["v"][::100] = float("inf")  # in every tile
    st = DeviceStatus()
    torch.cuda.synchronize()
    wait_limit(0)
    tree_attention(**sick, status=st)
    with pytest.raises(TimeoutError):
        st.check_status()
    wait_limit(-1)
    assert torch.equal(tree_attention(**args, status=st), want)
    st.check_status()


@pytest.mark.parametrize("case", [CASES[4], CASES[6], CASES[7], *CASES[13:19], CASES[22], *CASES[24:28]])
def test_attention_with_short_waits_is_right_or_says_so(case, wait_limit):
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    args, _ = _case(*case[:7], seed=4, kind=case[7])
    want, st = tree_attention(**args), DeviceStatus()
    for attempts in (0, 1, 2, 4, 16, 0):
        torch.cuda.synchronize()
        wait_limit(attempts)
        got = tree_attention(**args, status=st)
        try:
            st.check_status()
            assert torch.equal(got, want)
        except TimeoutError:
            pass
    wait_limit(-1)
    assert torch.equal(tree_attention(**args, status=st), want)
    st.check_status()


@pytest.mark.parametrize("group,batch", [(1, 12500), (16, 12500), (8, 12500), (1, 1)])  # 16, 128 (wide), 64 rows; wide with one head per key/value head
def test_attention_of_a_long_chain_with_values_that_are_not_finite(group, batch):
    """Two values that are not finite among 100000 nodes: looking for them at a row's end must not outlast the other warps' waits.

    Rows that see none of them, or only the first, are compared with the formula; the allowance is tree_util.attention's (see there).
    """
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import tree_attention

    n, dim = 100_000, 64
    g = torch.Generator(device="cuda").manual_seed(group)
    q, k, v = (torch.randn(n, h, dim, device="cuda", generator=g).to(torch.bfloat16) for h in (group, 1, 1))
    v[7, 0, 3], v[n - 9, 0, 5] = float("inf"), float("nan")
    cache = torch.zeros(1, 16, 1, dim, dtype=torch.bfloat16, device="cuda")
    starts = _i32([0] + [n] * batch)
    st = DeviceStatus()
    out = tree_attention(q, k, v, cache, cache, torch.zeros(batch, 1, dtype=torch.int32, device="cuda"), _i32([0] * batch), starts, status=st)
    st.check_status()
    clean = v.clone()
    clean[7, 0, 3] = clean[n - 9, 0, 5] = 0
    for i in (0, 6, 7, 500, 49_999, n - 10, n - 9, n - 1):
        # The last node of a chain of i + 1 nodes, as a tree of one node behind i cached ones: the plain form's single row.
        pad = -(i % -16)
        kc, vc = (torch.cat([x[:i], x.new_zeros(pad, 1, dim)]).view(-1, 16, 1, dim) for x in (k, clean))
        row = slice(i, i + 1)
        ref, _, tol, _ = U.attention(q[row], k[row], clean[row], kc, vc, [list(range(len(kc)))], [i], [0, 1], [None])
        bad = torch.zeros(group, dim, dtype=torch.bool, device="cuda")
        if i >= 7:
            assert (out[i, :, 3] == float("inf")).all()
            bad[:, 3] = True
        if i >= n - 9:
            assert out[i, :, 5].isnan().all()
            bad[:, 5] = True
        err = (out[i].double() - ref[0]).abs()
        assert bool((err <= tol[0])[~bad].all()), i


# ------------------------------------------------------------------------------------------------ the step as a whole
def _model(token, position, heads, dim):
    """Deterministic rows of a toy layer: one vector per (token, position)."""
    g = torch.Generator().manual_seed(int(token) * 4099 + int(position))
    return torch.randn(heads, dim, generator=g)


def test_one_step_end_to_end_and_replayed_from_a_graph():
    """Masks, attention, acceptance, tables and writes together, twice through one captured graph with new inputs:
    the cache then holds what a cache of the accepted tokens would, and the next step's attention reads it."""
    from actfold_b200.kernels import DeviceStatus
    from actfold_b200.speculative import accept_tree, block_tables, tree_attention, tree_masks, write_cache

    heads, kv, dim, page, keep, batch, n, layers = 4, 2, 64, 16, 5, 3, 12, 2
    rng = np.random.default_rng(0)
    pool, most = 40, 8
    kc = torch.full((layers, pool, page, kv, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    tables = torch.full((batch, most), -1, dtype=torch.int32, device="cuda")
    ring, span = _i32(rng.permutation(pool).tolist()), torch.tensor([0, pool], device="cuda")
    st = DeviceStatus()
    texts = [[int(x) for x in rng.integers(0, 50, m)] for m in (30, 1, 45)]

    def rows(tokens, positions, salt):
        return torch.stack([_model(t + 100 * salt, p, kv, dim) for t, p in zip(tokens, positions)]).to(torch.bfloat16).cuda()

    # Prompts: packed rows of every layer into their slots.
    lens = [len(t) for t in texts]
    step = block_tables(tables, _i32([0] * batch), _i32(lens), ring, span, page, sum(lens) + 2, status=st)
    flat, where = [x for t in texts for x in t], [p for t in texts for p in range(len(t))]
    for x, y in ((0, kc), (5, vc)):
        r = torch.stack([rows(flat, where, x + l) for l in range(layers)])
        if x == 0:
            kr = r
        else:
            write_cache(kr, r, kc, vc, step.slots[: len(flat)], status=st)
    span = step.free_range.clone()
    lengths, held = step.totals.clone(), step.totals.clone()
    # Static inputs of the captured step.
    parents, starts = _i32([-1] * (batch * n)), _i32([0, n, 2 * n, 3 * n])
    tokens, targets = (torch.zeros(batch * n, dtype=torch.int64, device="cuda") for _ in range(2))
    root = torch.zeros(batch, dtype=torch.int64, device="cuda")
    q = torch.zeros(batch * n, heads, dim, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(layers, batch * n, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def whole():
        mask, pos = tree_masks(parents, starts, 1, lengths, status=st)
        outs = [tree_attention(q, k[l], v[l], kc[l], vc[l], tables, lengths, starts, mask, status=st) for l in range(layers)]
        got = accept_tree(parents, tokens, targets, starts, keep, root, status=st)
        new = block_tables(tables, lengths, got.counts, ring, span, page, keep, held=held, padded=True, status=st)
        write_cache(k, v, kc, vc, new.slots, rows=got.rows, status=st)
        span.copy_(new.free_range)
        lengths.copy_(new.totals)
        held.copy_(new.totals)
        return mask, pos, outs, got

    side = torch.cuda.Stream()
    saved = [t.clone() for t in (kc, vc, tables, ring, span, lengths, held)]
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        whole()  # warm-up
    torch.cuda.synchronize()
    for t, s in zip((kc, vc, tables, ring, span, lengths, held), saved):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mask, pos, outs, got = whole()
    for t, s in zip((kc, vc, tables, ring, span, lengths, held), saved):
        t.copy_(s)
    for _ in range(4):
        trees = [U.random_parents(n, rng, chain=0.5) for _ in range(batch)]
        tok, tgt, rt = rng.integers(0, 2, batch * n), rng.integers(0, 2, batch * n), rng.integers(0, 2, batch)
        before = [len(t) for t in texts]
        depth = [len(p) - 1 for t in trees for p in U.ancestors(t)]
        where = [before[i // n] + d for i, d in enumerate(depth)]
        parents.copy_(_i32([p for t in trees for p in t]))
        tokens.copy_(torch.from_numpy(tok)), targets.copy_(torch.from_numpy(tgt)), root.copy_(torch.from_numpy(rt))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(int(tok.sum()))).cuda())
        for l in range(layers):
            k[l], v[l] = rows(tok, where, l), rows(tok, where, 5 + l)
        graph.replay()
        st.check_status()
        assert pos.tolist() == where
        # Attention against a dense cache of the texts.
        for l in range(layers):
            dk = torch.cat([rows(t, range(len(t)), l) for t in texts])
            dv = torch.cat([rows(t, range(len(t)), 5 + l) for t in texts])
            at = np.cumsum([0] + before)
            size = max(before) // page + 1
            pk, pv = (torch.zeros(batch * size, page, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            for b in range(batch):
                pk.view(batch, -1, kv, dim)[b, : before[b]], pv.view(batch, -1, kv, dim)[b, : before[b]] = dk[at[b]: at[b + 1]], dv[at[b]: at[b + 1]]
            bits = []
            for t in trees:
                m = torch.zeros(n, n, dtype=torch.bool)
                for i, p in enumerate(U.ancestors(t)):
                    m[i, p] = True
                bits.append(m)
            ref, _, tol, _ = U.attention(q, k[l], v[l], pk, pv, [list(range(b * size, (b + 1) * size)) for b in range(batch)], before, [0, n, 2 * n, 3 * n], bits)
            assert bool(((outs[l].double() - ref).abs() <= tol).all())
        for b, t in enumerate(trees):
            lo, hi = b * n, b * n + n
            path, nxt = U.accept(t, tok[lo:hi].tolist(), tgt[lo:hi].tolist(), int(rt[b]), keep)
            assert got.counts[b].item() == len(path) and got.next_tokens[b].item() == nxt
            texts[b] += [int(tok[lo + i]) for i in path]
        assert lengths.tolist() == [len(t) for t in texts]
        for b, t in enumerate(texts):
            for l in range(layers):
                pages = tables[b, : -(-len(t) // page)].long()
                assert torch.equal(kc[l][pages].flatten(0, 1)[: len(t)], rows(t, range(len(t)), l))
                assert torch.equal(vc[l][pages].flatten(0, 1)[: len(t)], rows(t, range(len(t)), 5 + l))
