"""Tree verification over a paged key/value cache: torch-facing wrappers of the C-ABI operators.

One step of speculative decoding for a batch of requests whose drafted tokens
form trees (actfold/speculative/branch_tree.py:11-95 keeps such a tree on the
host and verifies one branch per forward pass; here all nodes of all requests
are verified at once):

1. :func:`tree_masks` turns the parents of the drafted nodes into ancestor bits and positions;
2. :func:`tree_attention`, per layer, attends from every node to its request's cached prefix and its own ancestors;
3. :func:`accept_tree` keeps the longest path that agrees with the target model;
4. :func:`block_tables` hands out pages and slots for the kept tokens (or for a prompt's);
5. :func:`write_cache` writes the kept nodes' keys and values, of all layers at once, into their slots.

Nodes are packed: tree b holds nodes ``starts[b] .. starts[b + 1]`` and a
parent comes before its children. Sizes that change from step to step
(``starts``, lengths, counts) stay on the device, and no call synchronises, so a
step can be captured into a CUDA graph. Pass a
:class:`~actfold_b200.kernels.DeviceStatus` on the tensors' device to learn of values that the
kernels found out of range or out of capacity (``check_status()`` raises). Each call is ordered on
the current stream of its tensors' device; its scratch comes from torch's
allocator on that stream.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from actfold_b200 import _lib
from actfold_b200.kernels import DeviceStatus

_I32, _I64 = torch.int32, torch.int64
_ATTENTION = struct.Struct("3q2q2q2q2q3q3q2q3q2q3q6qd3q3q")
_ROWS = struct.Struct("2q3q3q2q4q4q2q7q")


class BlockTables(NamedTuple):
    """Result of :func:`block_tables` (device tensors)."""

    starts: torch.Tensor      # [requests + 1] int32: prefix sums of the new tokens
    totals: torch.Tensor      # [requests] int32: tokens that the tables now cover
    slots: torch.Tensor       # int64: page * page_size + offset of each new token, -1 elsewhere
    free_range: torch.Tensor  # [2] int64: the ring's free entries after the call


class AcceptedPath(NamedTuple):
    """Result of :func:`accept_tree` (device tensors)."""

    rows: torch.Tensor         # [trees, keep] int32: packed node numbers along the path, -1 behind the last
    counts: torch.Tensor       # [trees] int32
    next_tokens: torch.Tensor  # [trees] int64: the target model's choice after the path


# These calls are short, so what the host does per call counts: plain
# comparisons, no helper objects, and the stream's handle without a Stream object
# (where torch has these two names; it need not: one built without CUDA has neither).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.stream_ptr)


def _launch(what: str, index: int, fn, *args) -> None:
    if index == _current_device():
        st = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _current_stream(index))
    if st:
        _lib.check(st, what)


def _same_device(what: str, *tensors: torch.Tensor | None) -> int:
    """The index of the CUDA device that every given tensor is on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (index < 0 or t.get_device() != index):
            _lib.require_cuda(*tensors, what=what)
            raise ValueError(f"{what}: tensors are on {tensors[0].device} and {t.device}")
    return index


def _not_vectors(what: str, dtype: torch.dtype, **tensors: torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is not None and (t.dtype is not dtype or t.dim() != 1):
            raise ValueError(f"{what}: {name} must be a {dtype} vector, got {t.dtype} {tuple(t.shape)}")


def _word(status: DeviceStatus | None) -> torch.Tensor | None:
    return None if status is None else status.status


def block_tables(
    tables: torch.Tensor,
    lengths: torch.Tensor,
    grow: torch.Tensor,
    free_pages: torch.Tensor,
    free_range: torch.Tensor,
    page_size: int,
    slot_capacity: int,
    held: torch.Tensor | None = None,
    padded: bool = False,
    status: DeviceStatus | None = None,
) -> BlockTables:
    """Pages and slots for ``grow[r]`` new tokens behind the first ``lengths[r]`` tokens of every request.

    ``tables`` [requests, max_pages] int32 (updated in place) holds the pages
    of each request's first ``held[r]`` tokens (default: ``lengths``), each of one request only. Missing
    pages come from the front of the ring ``free_pages`` [pool] int32, pages no
    longer needed go to its end (updated in place). ``free_range`` [2] int64 holds the ring's
    first free entry and the one behind its last, counted without end (entry e
    lies at ``e % pool``); a ring with every page free starts as ``[0, pool]``.
    It is not changed: the new range is in the result. ``slots`` is
    [slot_capacity], packed at ``starts``, or with ``padded`` [requests,
    slot_capacity], -1 behind a request's last new token. Requests that do
    not fit leave everything as it was, with empty ``starts`` and -1 slots, and
    set the capacity bit of ``status``; so do, with the bounds bit, a negative number
    and a negative entry (no page) among those that would change hands. New tokens of a
    held page that is negative get slot -1 and set the bounds bit. The ring has at least one place.
    """
    if tables.dim() != 2 or tables.dtype is not _I32:
        raise ValueError(f"block_tables: tables must be int32 [requests, max_pages], got {tables.dtype} {tuple(tables.shape)}")
    n, most = tables.shape
    row, inner = tables.stride()
    if (inner != 1 and most > 1) or (row < most and n > 1):
        raise ValueError("block_tables: the rows of tables must be contiguous and must not overlap")
    if not (lengths.dtype is grow.dtype is free_pages.dtype is _I32 and lengths.dim() == grow.dim() == free_pages.dim() == 1
            and (held is None or (held.dtype is _I32 and held.dim() == 1))):
        _not_vectors("block_tables", _I32, lengths=lengths, grow=grow, held=held, free_pages=free_pages)
    if lengths.shape[0] != n or grow.shape[0] != n or (held is not None and held.shape[0] != n):
        raise ValueError(f"block_tables: lengths, grow and held must have one entry for each of {n} requests")
    if not free_pages.is_contiguous():
        raise ValueError("block_tables: free_pages must be contiguous")
    if free_range.dtype is not _I64 or free_range.shape != (2,):
        raise ValueError(f"block_tables: free_range must be two int64 numbers, got {free_range.dtype} {tuple(free_range.shape)}")
    if page_size <= 0 or slot_capacity < 0:
        raise ValueError(f"block_tables: page_size {page_size} must be positive and slot_capacity {slot_capacity} not negative")
    index = _same_device("block_tables", tables, lengths, grow, free_pages, free_range, held, word := _word(status))
    lengths, grow, free_range = lengths.contiguous(), grow.contiguous(), free_range.contiguous()
    if held is not None:
        held = held.contiguous()
    starts, totals, out = lengths.new_empty(n + 1), torch.empty_like(lengths), torch.empty_like(free_range)
    slots = free_range.new_empty((n, slot_capacity) if padded else slot_capacity)
    if n == 0:
        return BlockTables(starts.zero_(), totals, slots.fill_(-1), out.copy_(free_range))
    _launch("block_tables", index, _lib.load().af_block_tables, tables.data_ptr(), row if n > 1 else most, most,
            None if held is None else held.data_ptr(), lengths.data_ptr(), grow.data_ptr(), n, free_pages.data_ptr(), free_pages.shape[0],
            free_range.data_ptr(), page_size, n * slot_capacity if padded else slot_capacity, slot_capacity if padded else 0,
            starts.data_ptr(), totals.data_ptr(), slots.data_ptr(), out.data_ptr(), _lib.ptr(word))
    return BlockTables(starts, totals, slots, out)


def tree_masks(
    parents: torch.Tensor,
    starts: torch.Tensor,
    words: int,
    base: torch.Tensor | None = None,
    status: DeviceStatus | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Ancestor bits [nodes, words] int32 and positions [nodes] int32 of packed trees.

    ``parents`` [nodes] int32: number of a node's parent within its tree, -1
    for a node that follows the cached prefix. Bit ``j % 32`` of ``mask[i, j //
    32]`` is set for the node itself and its ancestors; ``positions[i] =
    base[b] + depth`` (``base`` = the prefix lengths). A tree may hold up to
    ``32 * words`` nodes. Rows behind ``starts[-1]`` are not written.
    """
    if not (parents.dtype is starts.dtype is _I32 and parents.dim() == starts.dim() == 1
            and (base is None or (base.dtype is _I32 and base.dim() == 1))):
        _not_vectors("tree_masks", _I32, parents=parents, starts=starts, base=base)
    batch, total = starts.shape[0] - 1, parents.shape[0]
    if batch < 0 or words <= 0:
        raise ValueError(f"tree_masks: starts needs one entry more than there are trees, words {words} must be positive")
    if base is not None and base.shape[0] != batch:
        raise ValueError(f"tree_masks: base must have one entry for each of {batch} trees")
    index = _same_device("tree_masks", parents, starts, base, word := _word(status))
    parents, starts = parents.contiguous(), starts.contiguous()
    if base is not None:
        base = base.contiguous()
    mask, positions = parents.new_empty((total, words)), torch.empty_like(parents)
    _launch("tree_masks", index, _lib.load().af_tree_masks, parents.data_ptr(), starts.data_ptr(), batch, total, words,
            None if base is None else base.data_ptr(), mask.data_ptr(), positions.data_ptr(), _lib.ptr(word))
    return mask, positions


def accept_tree(
    parents: torch.Tensor,
    tokens: torch.Tensor,
    targets: torch.Tensor,
    starts: torch.Tensor,
    keep: int,
    root_targets: torch.Tensor | None = None,
    max_nodes: int | None = None,
    status: DeviceStatus | None = None,
) -> AcceptedPath:
    """The longest path of each tree whose tokens the target model would have chosen.

    ``tokens`` [nodes] int64 are the drafted tokens, ``targets`` [nodes] int64
    the target model's choice after each node, ``root_targets`` [trees] its
    choice after the prefix (None: nodes that follow the prefix need no
    agreement). A node is accepted when its token is the choice after its
    parent and the parent is accepted. The deepest accepted node ends the path
    (of several, the one with the smallest number), which is cut to its first
    ``keep`` nodes. ``next_tokens`` is the choice after the last kept node
    (after the prefix when there is none, -1 when that is not given).
    ``max_nodes``: nodes of the largest tree, when known (at most 16384).
    """
    if not (parents.dtype is starts.dtype is _I32 and tokens.dtype is targets.dtype is _I64
            and parents.dim() == starts.dim() == tokens.dim() == targets.dim() == 1
            and (root_targets is None or (root_targets.dtype is _I64 and root_targets.dim() == 1))):
        _not_vectors("accept_tree", _I32, parents=parents, starts=starts)
        _not_vectors("accept_tree", _I64, tokens=tokens, targets=targets, root_targets=root_targets)
    batch, total = starts.shape[0] - 1, parents.shape[0]
    if tokens.shape[0] != total or targets.shape[0] != total:
        raise ValueError(f"accept_tree: tokens and targets must have one entry for each of {total} nodes")
    if batch < 0 or keep <= 0:
        raise ValueError(f"accept_tree: starts needs one entry more than there are trees, keep {keep} must be positive")
    if root_targets is not None and root_targets.shape[0] != batch:
        raise ValueError(f"accept_tree: root_targets must have one entry for each of {batch} trees")
    index = _same_device("accept_tree", parents, tokens, targets, starts, root_targets, word := _word(status))
    parents, tokens, targets, starts = parents.contiguous(), tokens.contiguous(), targets.contiguous(), starts.contiguous()
    if root_targets is not None:
        root_targets = root_targets.contiguous()
    rows, counts, following = parents.new_empty((batch, keep)), parents.new_empty(batch), tokens.new_empty(batch)
    _launch("accept_tree", index, _lib.load().af_accept_tree, parents.data_ptr(), tokens.data_ptr(), targets.data_ptr(), starts.data_ptr(),
            batch, total, 16384 if max_nodes is None else max_nodes, None if root_targets is None else root_targets.data_ptr(), keep,
            rows.data_ptr(), counts.data_ptr(), following.data_ptr(), _lib.ptr(word))
    return AcceptedPath(rows, counts, following)


def write_cache(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    rows: torch.Tensor | None = None,
    status: DeviceStatus | None = None,
) -> None:
    """Write key and value rows into their slots of a paged cache, in place.

    ``k``, ``v`` [n, kv_heads, dim] and caches [pages, page_size, kv_heads, dim], or both
    with a leading dimension of layers that share the slots. ``cache[slot // page_size, slot %
    page_size] = x[rows[i]]`` for each ``slot = slots[i]`` (``rows`` None: row
    i); entries with a negative slot or row are skipped. ``slots`` int64 and ``rows`` int32
    may have any shape, the same one. Any dtype, the caches' own; any strides but the
    innermost. Live slots must differ from one another, and the rows must not lie in the caches.
    """
    shape, cache = k.shape, k_cache.shape
    if v.shape != shape or v_cache.shape != cache or len(shape) not in (3, 4) or len(cache) != len(shape) + 1:
        raise ValueError(f"write_cache: k, v {tuple(k.shape)}, {tuple(v.shape)} do not match caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if len(shape) == 3:
        return write_cache(k[None], v[None], k_cache[None], v_cache[None], slots, rows, status)
    layers, n, heads, dim = shape
    if cache[0] != layers or cache[3] != heads or cache[4] != dim:
        raise ValueError(f"write_cache: rows {tuple(shape)} do not match caches {tuple(cache)}")
    dtype = k.dtype
    if v.dtype is not dtype or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"write_cache: rows {k.dtype}, {v.dtype} and caches {k_cache.dtype}, {v_cache.dtype} differ in dtype")
    if slots.dtype is not _I64 or (rows is not None and (rows.dtype is not _I32 or rows.shape != slots.shape)):
        raise ValueError("write_cache: slots must be int64, rows int32 of the same shape")
    count = slots.numel()
    if rows is None and count > n:
        raise ValueError(f"write_cache: {count} slots for {n} rows")
    if cache[2] == 0:
        raise ValueError("write_cache: page_size must be positive")
    kc0, kc1, kc2, kc3, kc4 = k_cache.stride()
    vc0, vc1, vc2, vc3, vc4 = v_cache.stride()
    if (kc4 != 1 or vc4 != 1) and dim > 1:
        raise ValueError("write_cache: the innermost dimension of the caches must be contiguous")
    if not (kc0 and kc1 and kc2 and kc3 and vc0 and vc1 and vc2 and vc3):
        if any(x == 0 and m > 1 for c in (k_cache, v_cache) for x, m in zip(c.stride(), cache)):
            raise ValueError("write_cache: the caches have entries that share memory")
    index = _same_device("write_cache", k, v, k_cache, v_cache, slots, rows, word := _word(status))
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if (k3 != 1 or v3 != 1) and dim > 1:
        k, v = k.contiguous(), v.contiguous()
        k0, k1, k2, k3 = v0, v1, v2, v3 = k.stride()
    slots = slots.contiguous()
    if rows is not None:
        rows = rows.contiguous()
    e = k.element_size()
    args = _ROWS.pack(k.data_ptr(), v.data_ptr(), e * k0, e * k1, e * k2, e * v0, e * v1, e * v2, k_cache.data_ptr(), v_cache.data_ptr(),
                      e * kc0, e * kc1, e * kc2, e * kc3, e * vc0, e * vc1, e * vc2, e * vc3, slots.data_ptr(),
                      0 if rows is None else rows.data_ptr(), n, count, cache[1], cache[2], layers, heads, dim * e)
    _launch("write_cache", index, _lib.load().af_write_cache, args, _lib.ptr(word))


def _grid(t: torch.Tensor) -> list[int] | None:
    """Strides in bytes of a 16-bit tensor (0 for a dimension of one entry), or None where its address or a stride is
    not a multiple of 16 bytes, the innermost dimension is not contiguous or entries share memory."""
    *outer, inner = t.stride()
    if inner != 1 or t.data_ptr() & 15:
        return None
    out = []
    for x, n in zip(outer, t.shape):
        if n == 1:
            x = 0
        elif x <= 0 or x & 7:
            return None
        out.append(2 * x)
    return out


def _row_grid(t: torch.Tensor) -> tuple | list | None:
    a, b, c = t.stride()
    return (2 * a, 2 * b) if c == 1 and a > 0 and b > 0 and not ((a | b) & 7 or t.data_ptr() & 15) else _grid(t)


def _cache_grid(t: torch.Tensor) -> tuple | list | None:
    a, b, c, d = t.stride()
    return (2 * a, 2 * b, 2 * c) if d == 1 and a > 0 and b > 0 and c > 0 and not ((a | b | c) & 7 or t.data_ptr() & 15) else _grid(t)


def tree_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    tables: torch.Tensor,
    lengths: torch.Tensor,
    starts: torch.Tensor,
    mask: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    status: DeviceStatus | None = None,
) -> torch.Tensor:
    """Attention of packed tree nodes over their requests' paged caches and their own trees.

    ``q`` [nodes, heads, dim], ``k`` / ``v`` [nodes, kv_heads, dim] of this
    step (not in the cache), caches [pages, page_size, kv_heads, dim] (any
    strides but the innermost, so a [pages, kv_heads, page_size, dim] cache is passed
    transposed), all fp16 or all bf16, dim 64 or 128, page_size a multiple of
    8. Request b's first ``lengths[b]`` tokens lie in pages ``tables[b]``;
    node i also sees the nodes whose bits are set in ``mask[i]`` ([nodes,
    words] int32, see :func:`tree_masks`; any bits are allowed, so a block that
    sees itself in both directions is a mask of ones). ``mask`` None: each
    tree is a chain, in which a node sees the nodes up to itself (a single new
    token, or a prompt behind a cached prefix; the work of a long one is that of a
    full square, about twice what its nodes see). ``scale`` defaults to dim **
    -0.5. A row that sees nothing is 0. ``lse`` [nodes, heads] float32 receives the
    natural log of each row's sum of exponentials. Rows of ``out`` behind ``starts[-1]`` are not written,
    none when ``starts`` is out of order. ``out`` shares no memory with the inputs.
    """
    qs, ks, cs = q.shape, k.shape, k_cache.shape
    if len(qs) != 3 or len(ks) != 3 or len(cs) != 4 or v.shape != ks or v_cache.shape != cs:
        raise ValueError(f"tree_attention: bad shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, caches "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    total, heads, dim = qs
    if ks[0] != total or ks[2] != dim or cs[2] != ks[1] or cs[3] != dim:
        raise ValueError(f"tree_attention: q {tuple(qs)}, k {tuple(ks)} and caches {tuple(cs)} do not match")
    dtype = q.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or k.dtype is not dtype or v.dtype is not dtype \
            or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"tree_attention: q, k, v and caches must all be fp16 or all bf16, got {q.dtype}, {k.dtype}, {v.dtype}, "
                         f"{k_cache.dtype}, {v_cache.dtype}")
    if tables.dim() != 2 or tables.dtype is not _I32:
        raise ValueError(f"tree_attention: tables must be int32 [requests, max_pages], got {tables.dtype} {tuple(tables.shape)}")
    batch, most = tables.shape
    if not (lengths.dtype is starts.dtype is _I32 and lengths.dim() == starts.dim() == 1):
        _not_vectors("tree_attention", _I32, lengths=lengths, starts=starts)
    if lengths.shape[0] != batch or starts.shape[0] != batch + 1:
        raise ValueError(f"tree_attention: {batch} requests need as many lengths and one entry of starts more")
    index = q.get_device()
    mask_at = mask_row = words = 0
    if mask is not None:
        if mask.dim() != 2 or mask.dtype is not _I32 or mask.shape[0] != total or mask.shape[1] == 0:
            raise ValueError(f"tree_attention: mask must be int32 [{total}, words], got {mask.dtype} {tuple(mask.shape)}")
        words = mask.shape[1]
        mask_row, inner = mask.stride()
        if (words > 1 and inner != 1) or mask_row < words:
            mask = mask.contiguous()
            mask_row = words
        mask_at = mask.data_ptr()
    k_grid, v_grid = _cache_grid(k_cache), _cache_grid(v_cache)
    if k_grid is None or v_grid is None:
        raise ValueError("tree_attention: the caches' innermost dimension must be contiguous, their other strides multiples of 16 bytes")
    out_grid = None
    if out is not None:
        if out.shape != qs or out.dtype is not dtype or (out_grid := _row_grid(out)) is None:
            raise ValueError("tree_attention: out must have q's shape and dtype, a contiguous innermost dimension and 16-byte strides")
    if lse is not None and (lse.shape != (total, heads) or lse.dtype is not torch.float32 or not lse.is_contiguous()):
        raise ValueError(f"tree_attention: lse must be contiguous float32 [{total}, {heads}]")
    _same_device("tree_attention", q, k, v, k_cache, v_cache, tables, lengths, starts, mask, out, lse, word := _word(status))
    if most > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    lengths, starts = lengths.contiguous(), starts.contiguous()
    if (q_grid := _row_grid(q)) is None:
        q = q.clone(memory_format=torch.contiguous_format)
        q_grid = _grid(q)
    if (kr_grid := _row_grid(k)) is None:
        k = k.clone(memory_format=torch.contiguous_format)
        kr_grid = _grid(k)
    if (vr_grid := _row_grid(v)) is None:
        v = v.clone(memory_format=torch.contiguous_format)
        vr_grid = _grid(v)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_grid = (2 * heads * dim, 2 * dim)
    size = _scratch.get(index) or _workspace_bytes(index)
    workspace = lengths.new_empty(size >> 2)
    args = _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q_grid, *kr_grid, *vr_grid, k_cache.data_ptr(), v_cache.data_ptr(), *k_grid, *v_grid,
        cs[0], cs[1], tables.data_ptr(), tables.stride(0) if batch > 1 else most, most, lengths.data_ptr(), starts.data_ptr(),
        mask_at, mask_row if total > 1 else words, words, batch, total, heads, ks[1], dim, _lib.DTYPE[dtype],
        dim ** -0.5 if scale is None else scale, out.data_ptr(), *out_grid, 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), size)
    _launch("tree_attention", index, _lib.load().af_tree_attention, args, _lib.ptr(word))
    return out


_scratch: dict[int, int] = {}  # bytes of scratch per device


def _workspace_bytes(index: int) -> int:
    n = C.c_int64()
    with torch.cuda.device(index):
        _lib.check(_lib.load().af_tree_attention_workspace_bytes(C.byref(n)), "tree_attention")
    _scratch[index] = (n.value + 15) & ~15
    return _scratch[index]
