"""Long requests in less memory: a paged key/value cache in 4 bits, windowed attention over it, and eviction.

Next to the 16-bit cache of :mod:`actfold_b200.tree_kernels`, with the same
pages, tables and slots (:func:`~actfold_b200.tree_kernels.block_tables` serves both):

* :class:`Int4Cache` holds keys and values in 4 bits, with a 16-bit scale and offset for every 32 dims:
  160 bytes a token and head of 128 dims instead of 512;
* :func:`write_cache_int4` and :func:`read_cache_int4` move rows into their slots and back;
* :func:`tree_attention_int4` is tree attention over it, with an optional sliding window and first tokens ("sinks") that stay visible;
* :func:`attention_weights` adds up the attention that every cached token is given, in either cache;
* :func:`evict_cache` keeps, of a request that has outgrown its budget, the tokens that were given the most, in either cache.

No call synchronises; sizes that change from step to step stay on the device,
so a step can be captured into a CUDA graph. Pass a
:class:`~actfold_b200.kernels.DeviceStatus` on the tensors' device to learn of
values that the kernels found out of range. Each call is ordered on the
current stream of its tensors' device; its scratch comes from torch's
allocator on that stream.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from actfold_b200 import _lib
from actfold_b200.kernels import DeviceStatus
from actfold_b200.tree_kernels import _grid, _launch, _not_vectors, _row_grid, _same_device, _word

_I32, _I64 = torch.int32, torch.int64
_CACHE = "q3q6q"
_ROWS = struct.Struct("2q3q3q2q2q" + _CACHE)
_ATTENTION = struct.Struct("3q2q2q2q" + _CACHE + "3q2q3q5qdq2qq2q")
_WEIGHTS = struct.Struct("q2q" + _CACHE + "q3q2q5qdqq2qq")
_EVICT = struct.Struct(_CACHE + "2q4q4q5q3q2qq3qq3q3q")
_NO_CACHE = (0,) * 10


class Int4Cache:
    """A paged key/value cache in 4 bits.

    ``data`` is uint8 [pages, kv_heads, page_size / 8, 10 * dim], or with a leading dimension of layers, dim 64 or 128; ``dtype``
    (fp16 or bf16) is that of the rows that go in and come out, and of the scales and offsets. Its last two dimensions are
    contiguous, its other strides multiples of 16 bytes. :meth:`empty` makes one; ``cache[l]`` is layer l. The pages hold what
    :func:`write_cache_int4` wrote; places that were never written are never used. ``data`` may be set
    to another tensor of the same layout, which all calls after that use; for any other make another cache.
    """

    __slots__ = ("_data", "dtype", "dim", "kv_heads", "pages", "page_size", "layers", "_packed")

    def __init__(self, data: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> None:
        shape = data.shape
        if data.dtype is not torch.uint8 or len(shape) not in (4, 5) or shape[-1] not in (640, 1280):
            raise ValueError(f"Int4Cache: data must be uint8 [(layers,) pages, kv_heads, page_size / 8, 640 or 1280], got {data.dtype} {tuple(shape)}")
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            raise ValueError(f"Int4Cache: dtype must be fp16 or bf16, got {dtype}")
        if len(shape) == 4:
            (pages, heads, blocks, size), layers = shape, None
            (sp, sh, sb, inner), sl = data.stride(), 0
        else:
            layers, pages, heads, blocks, size = shape
            sl, sp, sh, sb, inner = data.stride()
        if blocks == 0:
            raise ValueError("Int4Cache: page_size must be positive")
        if inner != 1 or (sb != size and blocks > 1):
            raise ValueError("Int4Cache: the blocks of a page's head must be contiguous")
        run = blocks * size
        if heads <= 1:
            sh = 0
        elif sh < run:
            raise ValueError("Int4Cache: data has entries that share memory")
        if pages <= 1:
            sp = 0
        elif sp < run:
            raise ValueError("Int4Cache: data has entries that share memory")
        if layers is not None and layers > 1:
            if sl < run:
                raise ValueError("Int4Cache: data has entries that share memory")
        else:
            sl = 0
        at = data.data_ptr()
        if (sl | sp | sh | at) & 15:
            raise ValueError("Int4Cache: data's address and strides must be multiples of 16 bytes")
        self._data, self.dtype, self.dim, self.layers, self.pages, self.kv_heads = data, dtype, size // 10, layers, pages, heads
        self.page_size = page = 8 * blocks
        self._packed = (at, sl, sp, sh, 1 if layers is None else layers, pages, page, heads, size // 10, _lib.DTYPE[dtype])

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @data.setter
    def data(self, data: torch.Tensor) -> None:
        old = self._data
        if data.dtype is not old.dtype or data.shape != old.shape or data.stride() != old.stride():
            raise ValueError(f"Int4Cache: data {data.dtype} {tuple(data.shape)} {data.stride()} has another layout than {tuple(old.shape)} {old.stride()}")
        self._data = data
        self._packed = (None, *self._packed[1:])

    def _at(self) -> tuple[int, ...]:
        """The cache as the C entry points take it, once ``data`` has been set to another tensor: its address is asked for when a call needs it."""
        if self._packed[0] is None:
            if (at := self._data.data_ptr()) & 15:
                raise ValueError("Int4Cache: data's address must be a multiple of 16 bytes")
            self._packed = (at, *self._packed[1:])
        return self._packed

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, dim: int, dtype: torch.dtype = torch.bfloat16, layers: int | None = None,
              device: torch.device | str = "cuda") -> "Int4Cache":
        """A cache with nothing in it."""
        if page_size <= 0 or page_size % 8 or dim not in (64, 128) or pages < 0 or kv_heads <= 0:
            raise ValueError(f"Int4Cache: page_size {page_size} must be a positive multiple of 8, dim {dim} 64 or 128, pages and kv_heads positive")
        shape = (pages, kv_heads, page_size // 8, 10 * dim)
        return cls(torch.empty(shape if layers is None else (layers, *shape), dtype=torch.uint8, device=device), dtype)

    def __getitem__(self, layer: int) -> "Int4Cache":
        if self.layers is None:
            raise ValueError("Int4Cache: the cache has no layers")
        return Int4Cache(self.data[layer], self.dtype)


class EvictedCache(NamedTuple):
    """Result of :func:`evict_cache` (device tensors)."""

    lengths: torch.Tensor  # [requests] int32: tokens that are left
    kept: torch.Tensor     # [(layers,) requests, kv_heads, keep] int32: the places that they came from, -1 behind the last
    weights: torch.Tensor  # like the call's weights: theirs, 0 behind the last


def _row_strides(t: torch.Tensor) -> tuple[int, int, int] | None:
    """Strides in bytes of 16-bit rows [layers, n, heads, dim], or None where they or the address are not multiples of 16."""
    a, b, c, d = t.stride()
    layers, n, heads, _ = t.shape
    a, b, c = 0 if layers <= 1 else 2 * a, 0 if n <= 1 else 2 * b, 0 if heads <= 1 else 2 * c
    return None if d != 1 or (a | b | c | t.data_ptr()) & 15 else (a, b, c)


def write_cache_int4(
    k: torch.Tensor,
    v: torch.Tensor,
    cache: Int4Cache,
    slots: torch.Tensor,
    rows: torch.Tensor | None = None,
    status: DeviceStatus | None = None,
) -> None:
    """Write key and value rows into their slots of a 4-bit cache, in place.

    ``k``, ``v`` [n, kv_heads, dim], or with the cache's leading dimension of layers that share the slots, of the cache's dtype
    and any strides. Entry i puts row ``rows[i]`` (``rows`` None: row i) into ``slots[i]`` (page * page_size + offset, as
    :func:`~actfold_b200.tree_kernels.block_tables` gives them); entries with a negative slot or row are skipped. ``slots`` int64
    and ``rows`` int32 may have any shape, the same one. Live slots must differ from one another. Of every 32 dims of a row the
    smallest value is kept as it is, the others lie within half a step of a fifteenth of their range (and the rounding to dtype);
    32 dims with a value that is not finite become NaN throughout.
    """
    layered = cache.layers is not None
    if v.shape != k.shape or k.dim() != (4 if layered else 3) or k.shape[-2:] != (cache.kv_heads, cache.dim) or (layered and k.shape[0] != cache.layers):
        raise ValueError(f"write_cache_int4: k, v {tuple(k.shape)}, {tuple(v.shape)} do not match a cache {tuple(cache.data.shape)}")
    if k.dtype is not cache.dtype or v.dtype is not cache.dtype:
        raise ValueError(f"write_cache_int4: rows {k.dtype}, {v.dtype} differ from the cache's {cache.dtype}")
    if slots.dtype is not _I64 or (rows is not None and (rows.dtype is not _I32 or rows.shape != slots.shape)):
        raise ValueError("write_cache_int4: slots must be int64, rows int32 of the same shape")
    if not layered:
        k, v = k[None], v[None]
    n, count = k.shape[1], slots.numel()
    if rows is None and count > n:
        raise ValueError(f"write_cache_int4: {count} slots for {n} rows")
    index = _same_device("write_cache_int4", k, v, cache.data, slots, rows, word := _word(status))
    if (ks := _row_strides(k)) is None:
        k = k.clone(memory_format=torch.contiguous_format)
        ks = _row_strides(k)
    if (vs := _row_strides(v)) is None:
        v = v.clone(memory_format=torch.contiguous_format)
        vs = _row_strides(v)
    slots = slots.contiguous()
    if rows is not None:
        rows = rows.contiguous()
    args = _ROWS.pack(k.data_ptr(), v.data_ptr(), *ks, *vs, slots.data_ptr(), 0 if rows is None else rows.data_ptr(), n, count, *cache._at())
    _launch("write_cache_int4", index, _lib.load().af_write_cache_int4, args, _lib.ptr(word))


def read_cache_int4(
    cache: Int4Cache,
    slots: torch.Tensor,
    status: DeviceStatus | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [(layers,) *slots.shape, kv_heads, dim] of the cache's dtype that lie in ``slots`` (int64; negative ones read as 0)."""
    if slots.dtype is not _I64:
        raise ValueError(f"read_cache_int4: slots must be int64, got {slots.dtype}")
    index = _same_device("read_cache_int4", cache.data, slots, word := _word(status))
    slots = slots.contiguous()
    shape = (*slots.shape, cache.kv_heads, cache.dim) if cache.layers is None else (cache.layers, *slots.shape, cache.kv_heads, cache.dim)
    k = torch.empty(shape, dtype=cache.dtype, device=slots.device)
    v = torch.empty_like(k)
    count, row = slots.numel(), 2 * cache.kv_heads * cache.dim
    st = (count * row, row, 2 * cache.dim)
    args = _ROWS.pack(k.data_ptr(), v.data_ptr(), *st, *st, slots.data_ptr(), 0, count, count, *cache._at())
    _launch("read_cache_int4", index, _lib.load().af_read_cache_int4, args, _lib.ptr(word))
    return k, v


def _check_tables(what: str, tables: torch.Tensor, lengths: torch.Tensor) -> tuple[int, int]:
    if tables.dim() != 2 or tables.dtype is not _I32:
        raise ValueError(f"{what}: tables must be int32 [requests, max_pages], got {tables.dtype} {tuple(tables.shape)}")
    if lengths.dtype is not _I32 or lengths.dim() != 1:
        _not_vectors(what, _I32, lengths=lengths)
    if lengths.shape[0] != tables.shape[0]:
        raise ValueError(f"{what}: lengths must have one entry for each of {tables.shape[0]} requests")
    return tables.shape


def evict_cache(
    cache: Int4Cache | tuple[torch.Tensor, torch.Tensor],
    tables: torch.Tensor,
    lengths: torch.Tensor,
    weights: torch.Tensor,
    keep: int,
    sinks: int = 0,
    recent: int = 0,
    status: DeviceStatus | None = None,
) -> EvictedCache:
    """Of every request with more than ``keep`` cached tokens, keep those that were given the most attention.

    ``cache`` is an :class:`Int4Cache` or the pair (k_cache, v_cache) of :func:`~actfold_b200.tree_kernels.write_cache` (any dtype),
    in both cases with or without a leading dimension of layers; ``weights`` float32 [(layers,) requests, kv_heads, places], as
    :func:`attention_weights` adds them up. For each layer, request and head by itself the first ``sinks`` tokens, the last
    ``recent`` and, of those between, the ones with the largest weights stay (equal weights: the earlier tokens; NaN counts as the
    largest), ``keep`` in all. They move, in their order, to the request's first ``keep`` places, in place, so lengths stay the
    same for all layers and heads. Other requests stay as they are, also those of a length that is none (it sets ``status``, and
    the result holds it, and all weights, as they were). The tables are not changed: a
    :func:`~actfold_b200.tree_kernels.block_tables` call with ``lengths`` the result's and ``held`` the old ones returns the pages.
    Keys are moved as they are, so they have to hold their positions (as rotated keys do); a window of
    :func:`tree_attention_int4` counts places. No page may lie in the tables of two requests, or twice in one.
    """
    packed = isinstance(cache, Int4Cache)
    if not packed:
        k_cache, v_cache = cache
        if k_cache.shape != v_cache.shape or k_cache.dtype is not v_cache.dtype or k_cache.dim() not in (4, 5):
            raise ValueError(f"evict_cache: caches {k_cache.dtype} {tuple(k_cache.shape)} and {v_cache.dtype} {tuple(v_cache.shape)} do not match")
        layered = k_cache.dim() == 5
        if not layered:
            k_cache, v_cache = k_cache[None], v_cache[None]
        layers, pages, page, heads, dim = k_cache.shape
        if page == 0:
            raise ValueError("evict_cache: page_size must be positive")
        e = k_cache.element_size()
        strides = []
        for t in (k_cache, v_cache):
            if t.stride(4) != 1 and dim > 1:
                raise ValueError("evict_cache: the innermost dimension of the caches must be contiguous")
            st = [0 if n <= 1 else s * e for n, s in zip(t.shape[:4], t.stride()[:4])]
            if any(s <= 0 and n > 1 for n, s in zip(t.shape[:4], st)):
                raise ValueError("evict_cache: the caches have entries that share memory")
            if any(s & 15 for s in st) or t.data_ptr() & 15 or dim * e & 15:
                raise ValueError("evict_cache: the caches' rows and strides must be multiples of 16 bytes")
            strides += st
        held = (k_cache, v_cache)
        parts = (*_NO_CACHE, k_cache.data_ptr(), v_cache.data_ptr(), *strides, layers, pages, page, heads, dim * e)
    else:
        layered, layers, heads = cache.layers is not None, 1 if cache.layers is None else cache.layers, cache.kv_heads
        held = (cache.data, None)
    n, most = _check_tables("evict_cache", tables, lengths)
    if weights.dtype is not torch.float32 or weights.dim() != (4 if layered else 3) or weights.shape[-3:-1] != (n, heads) \
            or (layered and weights.shape[0] != layers):
        raise ValueError(f"evict_cache: weights must be float32 [{'layers, ' if layered else ''}{n}, {heads}, places], got {weights.dtype} {tuple(weights.shape)}")
    if keep < 0 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"evict_cache: sinks {sinks} and recent {recent} must not be negative, and together not more than keep {keep}")
    index = _same_device("evict_cache", *held, tables, lengths, weights, word := _word(status))
    if packed:
        parts = (*cache._at(), *((0,) * 15))
    elif k_cache.numel() and k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("evict_cache: k_cache and v_cache share memory, whose rows would move twice")
    if most > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    lengths = lengths.contiguous()
    places = weights.shape[-1]
    if places > 1 and weights.stride(-1) != 1:
        weights = weights.contiguous()
    kept = lengths.new_empty((*weights.shape[:-1], keep))
    left, out = torch.empty_like(lengths), torch.empty(weights.shape, dtype=torch.float32, device=weights.device)
    if layers == 0 or heads == 0:
        return EvictedCache(torch.clamp(lengths, max=keep), kept, out)
    ws = weights.stride()
    args = _EVICT.pack(*parts, tables.data_ptr(), tables.stride(0) if n > 1 else most, most, lengths.data_ptr(), n, weights.data_ptr(),
                       *(ws[:3] if layered else (0, *ws[:2])), places, keep, sinks, recent, kept.data_ptr(), out.data_ptr(), left.data_ptr())
    _launch("evict_cache", index, _lib.load().af_evict_cache, args, _lib.ptr(word))
    return EvictedCache(left, kept, out)


def _check_window(what: str, window: int | None, sinks: int) -> int:
    """The window as the C entry points take it (0: none)."""
    if window is None:
        if sinks:
            raise ValueError(f"{what}: sinks need a window")
        return 0
    if window <= 0 or sinks < 0:
        raise ValueError(f"{what}: window {window} must be positive and sinks {sinks} not negative")
    return window


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, tuple | list]:
    """A copy of 16-bit rows [n, heads, dim] whose address and strides are multiples of 16 bytes, and these."""
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _row_grid(t)


def tree_attention_int4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cache: Int4Cache,
    tables: torch.Tensor,
    lengths: torch.Tensor,
    starts: torch.Tensor,
    mask: torch.Tensor | None = None,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    status: DeviceStatus | None = None,
) -> torch.Tensor:
    """Attention of packed tree nodes over their requests' 4-bit caches and their own trees.

    As :func:`~actfold_b200.tree_kernels.tree_attention` over what :func:`read_cache_int4` gives for the prefix: ``q`` [nodes,
    heads, dim], ``k`` / ``v`` [nodes, kv_heads, dim] of this step (16 bits, not in the cache), all of the cache's dtype;
    ``cache`` without layers, or one layer of it. Request b's first ``lengths[b]`` tokens lie in pages ``tables[b]``; node i also
    sees the nodes whose bits are set in ``mask[i]`` ([nodes, words] int32), without a mask the nodes of its chain up to itself.

    With a ``window`` a node that sees c nodes (itself among them) sees the last ``window - c`` tokens of the prefix (none where
    that is negative) and the prefix's first ``sinks`` tokens. A chain, which has no mask, goes on where the prefix ends: a node sees
    the last ``window`` tokens of prefix and chain, itself among them, and the request's first ``sinks`` tokens, of which the chain holds
    those that the prefix does not; so a prompt may be cut anywhere.
    Nodes that a mask shows stay visible whatever the window. Only pages with visible tokens are read.

    ``scale`` defaults to dim ** -0.5. A row that sees nothing is 0. ``lse`` [nodes, heads] float32 receives the natural log of
    each row's sum of exponentials, as :func:`attention_weights` takes it. Rows of ``out`` behind ``starts[-1]`` are not written,
    none when ``starts`` is out of order. ``out`` shares no memory with the inputs.
    """
    if cache.layers is not None:
        raise ValueError("tree_attention_int4: cache must be one layer (cache[l])")
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or ks[0] != qs[0] or ks[1] != cache.kv_heads or ks[2] != cache.dim or qs[2] != cache.dim:
        raise ValueError(f"tree_attention_int4: q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)} and cache {tuple(cache.data.shape)} do not match")
    total, heads, dim = qs
    dtype = cache.dtype
    if q.dtype is not dtype or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"tree_attention_int4: q, k, v must be of the cache's {dtype}, got {q.dtype}, {k.dtype}, {v.dtype}")
    batch, most = _check_tables("tree_attention_int4", tables, lengths)
    if starts.dtype is not _I32 or starts.dim() != 1:
        _not_vectors("tree_attention_int4", _I32, starts=starts)
    if starts.shape[0] != batch + 1:
        raise ValueError(f"tree_attention_int4: {batch} requests need one entry of starts more")
    window = _check_window("tree_attention_int4", window, sinks)
    mask_at = mask_row = words = 0
    if mask is not None:
        if mask.dim() != 2 or mask.dtype is not _I32 or mask.shape[0] != total or mask.shape[1] == 0:
            raise ValueError(f"tree_attention_int4: mask must be int32 [{total}, words], got {mask.dtype} {tuple(mask.shape)}")
        words = mask.shape[1]
        mask_row, inner = mask.stride()
        if (words > 1 and inner != 1) or mask_row < words:
            mask = mask.contiguous()
            mask_row = words
        mask_at = mask.data_ptr()
    out_grid = None
    if out is not None and (out.shape != qs or out.dtype is not dtype or (out_grid := _row_grid(out)) is None):
        raise ValueError("tree_attention_int4: out must have q's shape and dtype, a contiguous innermost dimension and 16-byte strides")
    if lse is not None and (lse.shape != (total, heads) or lse.dtype is not torch.float32 or not lse.is_contiguous()):
        raise ValueError(f"tree_attention_int4: lse must be contiguous float32 [{total}, {heads}]")
    index = _same_device("tree_attention_int4", q, k, v, cache.data, tables, lengths, starts, mask, out, lse, word := _word(status))
    if most > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    lengths, starts = lengths.contiguous(), starts.contiguous()
    if (q_grid := _row_grid(q)) is None:
        q, q_grid = _rows16(q)
    if (k_grid := _row_grid(k)) is None:
        k, k_grid = _rows16(k)
    if (v_grid := _row_grid(v)) is None:
        v, v_grid = _rows16(v)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_grid = (2 * heads * dim, 2 * dim)
    size = _scratch.get(index) or _workspace_bytes(index)
    workspace = lengths.new_empty(size >> 2)
    args = _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q_grid, *k_grid, *v_grid, *cache._at(), tables.data_ptr(),
        tables.stride(0) if batch > 1 else most, most, lengths.data_ptr(), starts.data_ptr(), mask_at, mask_row if total > 1 else words, words, batch, total,
        heads, window, sinks, dim ** -0.5 if scale is None else scale, out.data_ptr(), *out_grid, 0 if lse is None else lse.data_ptr(),
        workspace.data_ptr(), size)
    _launch("tree_attention_int4", index, _lib.load().af_tree_attention_int4, args, _lib.ptr(word))
    return out


def attention_weights(
    q: torch.Tensor,
    cache: Int4Cache | torch.Tensor,
    tables: torch.Tensor,
    lengths: torch.Tensor,
    starts: torch.Tensor,
    lse: torch.Tensor,
    weights: torch.Tensor,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
    status: DeviceStatus | None = None,
) -> torch.Tensor:
    """Add the attention that rows give to every cached token to ``weights``, in place; returns ``weights``.

    ``weights`` float32 [requests, kv_heads, places]: entry (b, h, p) grows by the sum, over request b's rows and the query heads
    of group h, of ``exp(scale * q . k_p - lse)`` for the places p < ``lengths[b]`` that the row sees. ``q`` [nodes, heads, dim]
    and ``lse`` float32 [nodes, heads], as :func:`~actfold_b200.tree_kernels.tree_attention` or :func:`tree_attention_int4` left
    them for these rows; request b's rows ``starts[b] .. starts[b + 1]`` follow one another (one token, the accepted path of a tree,
    a prompt's next piece), and ``lengths``, ``window``, ``sinks`` and ``scale`` are that call's: of the tokens cached before the rows.
    What rows give to one another is not counted. A prompt over an empty cache adds nothing; in pieces, every piece adds to
    those before it. ``cache`` is one layer: an :class:`Int4Cache` or a 16-bit k_cache [pages, page_size, kv_heads, dim], page_size a
    multiple of 8, dim 64 or 128 (``window`` and ``sinks`` are there for rows whose attention had them; ``tree_attention`` has none).
    :func:`evict_cache` takes the weights.
    """
    packed = isinstance(cache, Int4Cache)
    if packed:
        if cache.layers is not None:
            raise ValueError("attention_weights: cache must be one layer (cache[l])")
        keys, dtype, kv, dim, token = cache.data, cache.dtype, cache.kv_heads, cache.dim, 0
    else:
        if cache.dim() != 4 or cache.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"attention_weights: cache must be an Int4Cache or 16-bit [pages, page_size, kv_heads, dim], got {cache.dtype} {tuple(cache.shape)}")
        pages, page, kv, dim = cache.shape
        if page == 0 or page % 8 or dim not in (64, 128) or kv == 0:
            raise ValueError(f"attention_weights: page_size {page} must be a positive multiple of 8, dim {dim} 64 or 128")
        if (grid := _grid(cache)) is None:
            raise ValueError("attention_weights: the cache's innermost dimension must be contiguous, its other strides multiples of 16 bytes")
        keys, dtype = cache, cache.dtype
        parts, token = (cache.data_ptr(), 0, grid[0], grid[2], 1, pages, page, kv, dim, _lib.DTYPE[dtype]), grid[1]
    qs = q.shape
    total, heads = (qs[0], qs[1]) if len(qs) == 3 else (0, 0)
    if heads == 0 or kv == 0 or q.dtype is not dtype or qs[2] != dim or heads % kv:
        raise ValueError(f"attention_weights: q {q.dtype} {tuple(qs)} and cache {dtype} {tuple(keys.shape)} do not match")
    batch, most = _check_tables("attention_weights", tables, lengths)
    if starts.dtype is not _I32 or starts.dim() != 1:
        _not_vectors("attention_weights", _I32, starts=starts)
    if starts.shape[0] != batch + 1:
        raise ValueError(f"attention_weights: {batch} requests need one entry of starts more")
    if lse.dtype is not torch.float32 or lse.shape != (total, heads):
        raise ValueError(f"attention_weights: lse must be float32 [{total}, {heads}], got {lse.dtype} {tuple(lse.shape)}")
    if weights.dtype is not torch.float32 or weights.dim() != 3 or weights.shape[:2] != (batch, kv):
        raise ValueError(f"attention_weights: weights must be float32 [{batch}, {kv}, places], got {weights.dtype} {tuple(weights.shape)}")
    places = weights.shape[2]
    w_request, w_head, inner = weights.stride()
    if (places > 1 and inner != 1) or (w_request == 0 and batch > 1) or (w_head == 0 and kv > 1):
        raise ValueError("attention_weights: the innermost dimension of weights must be contiguous, and its entries must not share memory")
    window = _check_window("attention_weights", window, sinks)
    index = _same_device("attention_weights", q, keys, tables, lengths, starts, lse, weights, word := _word(status))
    if packed:
        parts = cache._at()
    if most > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    lengths, starts, lse = lengths.contiguous(), starts.contiguous(), lse.contiguous()
    if (q_grid := _row_grid(q)) is None:
        q, q_grid = _rows16(q)
    args = _WEIGHTS.pack(q.data_ptr(), *q_grid, *parts, token, tables.data_ptr(), tables.stride(0) if batch > 1 else most, most, lengths.data_ptr(),
                         starts.data_ptr(), batch, total, heads, window, sinks, dim ** -0.5 if scale is None else scale, lse.data_ptr(),
                         weights.data_ptr(), w_request, w_head, places)
    _launch("attention_weights", index, _lib.load().af_attention_weights, args, _lib.ptr(word))
    return weights


_scratch: dict[int, int] = {}  # bytes of scratch per device


def _workspace_bytes(index: int) -> int:
    n = C.c_int64()
    with torch.cuda.device(index):
        _lib.check(_lib.load().af_tree_attention_int4_workspace_bytes(C.byref(n)), "tree_attention_int4")
    _scratch[index] = (n.value + 15) & ~15
    return _scratch[index]
