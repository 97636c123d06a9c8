"""What the 4-bit cache's operators hand to the library, at the edges of what their inputs may be (CPU only)."""

from __future__ import annotations

import pytest
import torch

from actfold_b200 import _lib
from actfold_b200 import cache_kernels as K
from actfold_b200 import speculative as S
from test_cache_kernels_host import _attention, _cache, _evict, _weights, _z, lib  # noqa: F401 (lib: a fixture)

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture
def launched(monkeypatch, lib):  # noqa: F811
    """The packed arguments of the calls, which go no further."""
    calls = []
    monkeypatch.setattr(K, "_same_device", lambda *a: 0)
    monkeypatch.setattr(K, "_launch", lambda what, index, fn, args, status: calls.append(args))
    monkeypatch.setattr(K, "_scratch", {0: 64})
    return calls


def _calls(cache):
    """Every operator that takes the cache, and where in its arguments the cache's numbers begin."""
    k, slots = _z(3, 2, 64, dtype=BF), _z(3, dtype=torch.int64)
    return ((lambda: S.write_cache_int4(k, k, cache, slots), K._ROWS, 12), (lambda: S.read_cache_int4(cache, slots), K._ROWS, 12),
            (lambda: S.tree_attention_int4(**_attention(cache=cache)), K._ATTENTION, 9), (lambda: S.attention_weights(**_weights(cache=cache)), K._WEIGHTS, 3),
            (lambda: S.evict_cache(**_evict(cache=cache)), K._EVICT, 0))


def test_calls_use_the_tensor_that_data_is_now(launched):
    """No call reads or writes memory that the cache had before: it may have been freed."""
    cache = _cache()
    old = cache.data
    for call, _, _ in _calls(cache):
        call()
    cache.data = new = _z(3, 2, 2, 640, dtype=torch.uint8)
    for call, _, _ in _calls(cache):
        call()
    for i, (_, struct, at) in enumerate(_calls(cache)):
        assert struct.unpack(launched[i])[at] == old.data_ptr()
        fields = struct.unpack(launched[i + 5])[at:at + 10]
        assert fields == (new.data_ptr(), 0, 2560, 1280, 1, 3, 16, 2, 64, _lib.DTYPE[BF])
    assert cache.data is new


def test_data_keeps_its_layout(launched):
    cache = _cache()
    held = cache.data
    u8 = torch.uint8
    for bad in (_z(3, 2, 2, 640), _z(5, 2, 2, 640, dtype=u8), _z(1, 3, 2, 2, 640, dtype=u8), _z(3, 2, 2, 1280, dtype=u8), _z(3, 2, 4, 640, dtype=u8)[:, :, ::2],
                _z(2, 3, 2, 640, dtype=u8).transpose(0, 1), _z(1, 2, 2, 640, dtype=u8).expand(3, 2, 2, 640)):
        with pytest.raises(ValueError, match="Int4Cache"):
            cache.data = bad
    assert cache.data is held
    cache.data = _z(3 * 2 * 2 * 640 + 16, dtype=u8)[8:-8].view(3, 2, 2, 640)  # not on a 16-byte border
    for call, _, _ in _calls(cache):
        with pytest.raises(ValueError, match="16 bytes"):
            call()
    assert not launched


def test_entries_that_share_memory_are_refused(launched, lib):  # noqa: F811
    """A page's head is one run of blocks: entries nearer to one another than that overlap, and may run past the tensor's end as read."""
    u8 = _z(4 * 3 * 2 * 4 * 640, dtype=torch.uint8)
    for shape, strides in (((3, 2, 4, 640), (2 * 2560, 1280, 640, 1)), ((3, 2, 4, 640), (640, 3 * 2560, 640, 1)), ((4, 3, 2, 4, 640), (2544, 5120, 2560, 640, 1))):
        with pytest.raises(ValueError, match="share memory"):
            S.Int4Cache(u8.as_strided(shape, strides))
    for shape, strides in (((3, 2, 4, 640), (2560, 3 * 2560, 640, 1)), ((1, 1, 4, 640), (16, 16, 640, 1)), ((1, 3, 2, 4, 640), (16, 5120, 2560, 640, 1))):
        S.Int4Cache(u8.as_strided(shape, strides))
    good = (u8.data_ptr() + 15 & ~15, 1 << 20, 5120, 2560, 2, 3, 32, 2, 64, _lib.DTYPE[BF])
    p = good[0]
    rows = lambda c: K._ROWS.pack(p, p, *(0, 256, 128) * 2, p, 0, 1, 1, *c)
    evict = lambda c: K._EVICT.pack(*c, *(0,) * 15, p, 2, 2, p, 1, p, 0, 64, 32, 32, 20, 0, 0, p, p, p)
    attention = lambda c: K._ATTENTION.pack(p, p, p, 256, 128, 128, 64, 128, 64, *c, p, 2, 2, p, p, 0, 0, 0, 1, 1, 2, 0, 0, 0.1, p, 256, 128, 0, p, 1 << 40)
    weights = lambda c, token=0: K._WEIGHTS.pack(p, 256, 128, *c, token, p, 2, 2, p, p, 1, 1, 2, 0, 0, 0.1, p, p, 64, 32, 32)
    for i in (1, 2, 3):
        near = (*good[:i], 2544, *good[i + 1:])
        calls = [(lib.af_write_cache_int4, rows), (lib.af_read_cache_int4, rows), (lib.af_evict_cache, evict)]
        for fn, pack in calls + ([] if i == 1 else [(lib.af_tree_attention_int4, attention), (lib.af_attention_weights, weights)]):
            assert fn(pack(near), None, None) == _lib.AF_ERR_ARG, (fn, i)
            assert b"share" in lib.af_last_error_string()
    # Rows of 16 bits whose tokens share one: no blocks of 4 bits, and no such rows either.
    for token in (0, -256):
        assert lib.af_attention_weights(weights((p, 0, 4096, 128, 1, 3, 32, 2, 64, good[9]), token), None, None) == _lib.AF_ERR_ARG


def test_a_cache_without_heads():
    """Calls that need query heads for it are refused."""
    cache = S.Int4Cache(_z(3, 0, 2, 640, dtype=torch.uint8))
    with pytest.raises(ValueError, match="attention_weights"):
        S.attention_weights(**_weights(cache=cache, weights=_z(2, 0, 40, dtype=torch.float32)))


def test_one_cache_for_keys_and_values_is_not_moved_twice(launched):
    """Keys and values are moved by CTAs that do not wait for one another."""
    rows = _z(3, 2, 16, 2, 64, dtype=BF)
    S.evict_cache(**_evict(cache=(rows[:, 0], rows[:, 1])))
    assert len(launched) == 1
    for one in (rows[:, 0], rows[None, :, 0]):
        with pytest.raises(ValueError, match="share memory"):
            S.evict_cache(**_evict(cache=(one, one), weights=_z(*one.shape[:-4], 2, 2, 40, dtype=torch.float32)))
    assert len(launched) == 1
