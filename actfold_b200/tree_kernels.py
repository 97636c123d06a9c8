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
:class:`~actfold_b200.kernels.DeviceStatus` to learn of values that the device
found out of range or out of capacity (``check_status()`` raises). Each call is ordered on
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


def _call(what: str, device: torch.device, fn, *args) -> None:
    if device.index == torch.cuda.current_device():
        st = fn(*args, _lib.stream_ptr(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _lib.stream_ptr(device))
    if st:
        _lib.check(st, what)


def _vector(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, n: int | None = None) -> torch.Tensor:
    if t.dim() != 1 or t.dtype is not dtype or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what}: {name} must be a {dtype} vector{'' if n is None else f' of {n}'}, got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _on_device(what: str, *tensors: torch.Tensor | None) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            _lib.require_cuda(t, what=what)
        if t.device != dev:
            raise ValueError(f"{what}: tensors are on {dev} and {t.device}")
    return dev


def _status(status: DeviceStatus | None) -> int | None:
    return None if status is None else status.status.data_ptr()


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
    of each request's first ``held[r]`` tokens (default: ``lengths``). Missing
    pages come from the front of the ring ``free_pages`` [pool] int32, pages no
    longer needed go to its end (updated in place). ``free_range`` [2] int64 holds the ring's
    first free entry and the one behind its last, counted without end (entry e
    lies at ``e % pool``); a ring with every page free starts as ``[0, pool]``.
    It is not changed: the new range is in the result. ``slots`` is
    [slot_capacity], packed at ``starts``, or with ``padded`` [requests,
    slot_capacity], -1 behind a request's last new token. Requests that do
    not fit leave everything as it was, with empty ``starts`` and -1 slots, and
    set the capacity bit of ``status``.
    """
    if tables.dim() != 2 or tables.dtype is not _I32 or (tables.shape[1] > 1 and tables.stride(1) != 1) or \
            (tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]):
        raise ValueError(f"block_tables: tables must be int32 [requests, max_pages] with contiguous rows, got {tables.dtype} {tuple(tables.shape)}")
    n, most = tables.shape
    lengths = _vector("block_tables", "lengths", lengths, _I32, n)
    grow = _vector("block_tables", "grow", grow, _I32, n)
    if held is not None:
        held = _vector("block_tables", "held", held, _I32, n)
    if free_pages.dim() != 1 or free_pages.dtype is not _I32 or not free_pages.is_contiguous():
        raise ValueError("block_tables: free_pages must be a contiguous int32 vector")
    free_range = _vector("block_tables", "free_range", free_range, _I64, 2)
    if page_size <= 0 or slot_capacity < 0:
        raise ValueError(f"block_tables: page_size {page_size} and slot_capacity {slot_capacity} must be positive")
    dev = _on_device("block_tables", tables, lengths, grow, free_pages, free_range, held)
    small = torch.empty(2 * n + 1, dtype=_I32, device=dev)
    slots = torch.empty((n, slot_capacity) if padded else slot_capacity, dtype=_I64, device=dev)
    out = torch.empty(2, dtype=_I64, device=dev)
    if n == 0:
        out.copy_(free_range)
        return BlockTables(small.zero_(), small[1:], slots.fill_(-1), out)
    at = small.data_ptr()
    _call("block_tables", dev, _lib.load().af_block_tables, tables.data_ptr(), tables.stride(0) if n > 1 else most, most,
          None if held is None else held.data_ptr(), lengths.data_ptr(), grow.data_ptr(), n, free_pages.data_ptr(), free_pages.shape[0],
          free_range.data_ptr(), page_size, n * slot_capacity if padded else slot_capacity, slot_capacity if padded else 0,
          at, at + 4 * (n + 1), slots.data_ptr(), out.data_ptr(), _status(status))
    starts, totals = small.split((n + 1, n))
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
    parents = _vector("tree_masks", "parents", parents, _I32)
    starts = _vector("tree_masks", "starts", starts, _I32)
    batch, total = starts.shape[0] - 1, parents.shape[0]
    if batch < 0 or words <= 0:
        raise ValueError(f"tree_masks: starts needs one entry more than there are trees, words {words} must be positive")
    if base is not None:
        base = _vector("tree_masks", "base", base, _I32, batch)
    dev = _on_device("tree_masks", parents, starts, base)
    mask = torch.empty((total, words), dtype=_I32, device=dev)
    positions = torch.empty(total, dtype=_I32, device=dev)
    _call("tree_masks", dev, _lib.load().af_tree_masks, parents.data_ptr(), starts.data_ptr(), batch, total, words,
          None if base is None else base.data_ptr(), mask.data_ptr(), positions.data_ptr(), _status(status))
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
    parents = _vector("accept_tree", "parents", parents, _I32)
    total = parents.shape[0]
    tokens = _vector("accept_tree", "tokens", tokens, _I64, total)
    targets = _vector("accept_tree", "targets", targets, _I64, total)
    starts = _vector("accept_tree", "starts", starts, _I32)
    batch = starts.shape[0] - 1
    if batch < 0 or keep <= 0:
        raise ValueError(f"accept_tree: starts needs one entry more than there are trees, keep {keep} must be positive")
    if root_targets is not None:
        root_targets = _vector("accept_tree", "root_targets", root_targets, _I64, batch)
    dev = _on_device("accept_tree", parents, tokens, targets, starts, root_targets)
    rows = torch.empty((batch, keep), dtype=_I32, device=dev)
    counts = torch.empty(batch, dtype=_I32, device=dev)
    following = torch.empty(batch, dtype=_I64, device=dev)
    _call("accept_tree", dev, _lib.load().af_accept_tree, parents.data_ptr(), tokens.data_ptr(), targets.data_ptr(), starts.data_ptr(),
          batch, total, 16384 if max_nodes is None else max_nodes, None if root_targets is None else root_targets.data_ptr(), keep,
          rows.data_ptr(), counts.data_ptr(), following.data_ptr(), _status(status))
    return AcceptedPath(rows, counts, following)


def _strides(t: torch.Tensor, scale: int) -> list[int]:
    """Strides in bytes, 0 for a dimension of one entry (torch leaves any value there)."""
    return [0 if n == 1 else s * scale for n, s in zip(t.shape[:-1], t.stride())]


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
    innermost. Live slots must differ from one another.
    """
    if k.shape != v.shape or k_cache.shape != v_cache.shape or k.dim() not in (3, 4) or k_cache.dim() != k.dim() + 1:
        raise ValueError(f"write_cache: k, v {tuple(k.shape)}, {tuple(v.shape)} do not match caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k.dim() == 3:
        k, v, k_cache, v_cache = k[None], v[None], k_cache[None], v_cache[None]
    layers, n, heads, dim = k.shape
    pages, page_size = k_cache.shape[1:3]
    if k_cache.shape[0] != layers or k_cache.shape[3:] != k.shape[2:]:
        raise ValueError(f"write_cache: rows {tuple(k.shape)} do not match caches {tuple(k_cache.shape)}")
    if not (k.dtype == v.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError(f"write_cache: rows {k.dtype}, {v.dtype} and caches {k_cache.dtype}, {v_cache.dtype} differ in dtype")
    if slots.dtype is not _I64 or (rows is not None and (rows.dtype is not _I32 or rows.shape != slots.shape)):
        raise ValueError("write_cache: slots must be int64, rows int32 of the same shape")
    if rows is None and slots.numel() > n:
        raise ValueError(f"write_cache: {slots.numel()} slots for {n} rows")
    if page_size == 0:
        raise ValueError("write_cache: page_size must be positive")
    if dim > 1 and (k_cache.stride(-1) != 1 or v_cache.stride(-1) != 1):
        raise ValueError("write_cache: the innermost dimension of the caches must be contiguous")
    for c in (k_cache, v_cache):
        if any(s == 0 and m > 1 for s, m in zip(c.stride(), c.shape)):
            raise ValueError("write_cache: the caches have entries that share memory")
    if dim > 1 and k.stride(-1) != 1:
        k = k.contiguous()
    if dim > 1 and v.stride(-1) != 1:
        v = v.contiguous()
    slots = slots.contiguous()
    rows = None if rows is None else rows.contiguous()
    dev = _on_device("write_cache", k, v, k_cache, v_cache, slots, rows)
    es = k.element_size()
    args = _ROWS.pack(k.data_ptr(), v.data_ptr(), *_strides(k, es), *_strides(v, es), k_cache.data_ptr(), v_cache.data_ptr(),
                      *_strides(k_cache, es), *_strides(v_cache, es), slots.data_ptr(), 0 if rows is None else rows.data_ptr(), n,
                      slots.numel(), pages, page_size, layers, heads, dim * es)
    _call("write_cache", dev, _lib.load().af_write_cache, args, _status(status))


def _aligned(t: torch.Tensor) -> bool:
    """Innermost dimension contiguous, address and strides multiples of 16 bytes."""
    if t.stride(-1) != 1 or t.data_ptr() & 15:
        return False
    unit = 16 // t.element_size()
    return all(n == 1 or (s > 0 and s % unit == 0) for n, s in zip(t.shape[:-1], t.stride()))


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
    token, or a prompt behind a cached prefix). ``scale`` defaults to dim **
    -0.5. A row that sees nothing is 0. ``lse`` [nodes, heads] float32 receives the
    natural log of each row's sum of exponentials. Rows of ``out`` behind ``starts[-1]`` are not written.
    """
    if q.dim() != 3 or k.dim() != 3 or k_cache.dim() != 4 or k.shape != v.shape or k_cache.shape != v_cache.shape:
        raise ValueError(f"tree_attention: bad shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, caches "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    total, heads, dim = q.shape
    kv_heads = k.shape[1]
    pages, page_size = k_cache.shape[:2]
    if k.shape[0] != total or k.shape[2] != dim or k_cache.shape[2] != kv_heads or k_cache.shape[3] != dim:
        raise ValueError(f"tree_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and caches {tuple(k_cache.shape)} do not match")
    if q.dtype not in (torch.float16, torch.bfloat16) or not (q.dtype == k.dtype == v.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError(f"tree_attention: q, k, v and caches must all be fp16 or all bf16, got {q.dtype}, {k.dtype}, {v.dtype}, "
                         f"{k_cache.dtype}, {v_cache.dtype}")
    if tables.dim() != 2 or tables.dtype is not _I32:
        raise ValueError(f"tree_attention: tables must be int32 [requests, max_pages], got {tables.dtype} {tuple(tables.shape)}")
    batch, most = tables.shape
    if most > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    lengths = _vector("tree_attention", "lengths", lengths, _I32, batch)
    starts = _vector("tree_attention", "starts", starts, _I32, batch + 1)
    words = 0
    if mask is not None:
        if mask.dim() != 2 or mask.dtype is not _I32 or mask.shape[0] != total or mask.shape[1] == 0:
            raise ValueError(f"tree_attention: mask must be int32 [{total}, words], got {mask.dtype} {tuple(mask.shape)}")
        words = mask.shape[1]
        if (words > 1 and mask.stride(1) != 1) or (total > 1 and mask.stride(0) < words):
            mask = mask.contiguous()
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or not _aligned(out)):
        raise ValueError("tree_attention: out must have q's shape and dtype, a contiguous innermost dimension and 16-byte strides")
    if lse is not None and (lse.shape != (total, heads) or lse.dtype is not torch.float32 or not lse.is_contiguous()):
        raise ValueError(f"tree_attention: lse must be contiguous float32 [{total}, {heads}]")
    if not (_aligned(k_cache) and _aligned(v_cache)):
        raise ValueError("tree_attention: the caches' innermost dimension must be contiguous, their other strides multiples of 16 bytes")
    dev = _on_device("tree_attention", q, k, v, k_cache, v_cache, tables, lengths, starts, mask, out, lse)
    q, k, v = (t if _aligned(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    if out is None:
        out = torch.empty((total, heads, dim), dtype=q.dtype, device=dev)
    lib = _lib.load()
    size = _workspace_bytes(dev)
    workspace = torch.empty(size, dtype=torch.uint8, device=dev)
    args = _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q, 2), *_strides(k, 2), *_strides(v, 2), k_cache.data_ptr(), v_cache.data_ptr(),
        *_strides(k_cache, 2), *_strides(v_cache, 2), pages, page_size, tables.data_ptr(), tables.stride(0) if batch > 1 else most, most,
        lengths.data_ptr(), starts.data_ptr(), 0 if mask is None else mask.data_ptr(), words if total == 1 or mask is None else mask.stride(0), words,
        batch, total, heads, kv_heads, dim, _lib.DTYPE[q.dtype], dim ** -0.5 if scale is None else float(scale),
        out.data_ptr(), *_strides(out, 2), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), size)
    _call("tree_attention", dev, lib.af_tree_attention, args, _status(status))
    return out


_scratch: dict[torch.device, int] = {}


def _workspace_bytes(device: torch.device) -> int:
    size = _scratch.get(device)
    if size is None:
        n = C.c_int64()
        with torch.cuda.device(device):
            _lib.check(_lib.load().af_tree_attention_workspace_bytes(C.byref(n)), "tree_attention")
        size = _scratch[device] = n.value
    return size
