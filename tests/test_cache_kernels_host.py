"""Refusals of the 4-bit cache's operators, and their plain forms against hand-made answers (CPU only)."""

from __future__ import annotations

import ctypes as C
import math
import os

import pytest
import torch

import cache_util as U
from actfold_b200 import _lib
from actfold_b200 import cache_kernels as K
from actfold_b200 import speculative as S

BF, HF = torch.bfloat16, torch.float16


def _z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _cache(pages=3, heads=2, blocks=2, dim=64, dtype=BF, layers=None):
    shape = (pages, heads, blocks, 10 * dim)
    return S.Int4Cache(_z(*(shape if layers is None else (layers, *shape)), dtype=torch.uint8), dtype)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from actfold_b200.build import build

        build()
    return _lib.load()


def test_plain_forms():
    x = torch.cat([torch.arange(32.0) / 2, torch.full((32,), 3.0)]).to(HF)
    codes, scales, offsets = U.encode(x[None])
    assert offsets.tolist() == [[0.0, 3.0]] and scales[0, 1] == 0 and codes[0, 32:].eq(0).all() and codes[0, 0] == 0 and codes[0, 31] == 15
    assert torch.equal(U.values(codes, scales, offsets)[0, 32:], x[32:])
    data = _z(2, 1, 1, 640, dtype=torch.uint8)
    U.put(data, 10, 1, codes, scales, offsets)  # page 1, row 2, values
    got = U.decoded(data, HF)
    assert torch.equal(got[1, 10, 0], U.values(codes, scales, offsets)[0]) and not got[0].any() and not got[1, :10].any()
    # A word holds dims 8 w + 2 i in its low half, 8 w + 2 i + 1 in its high one.
    row = data[1, 0, 0, 320 + 64: 320 + 68].tolist()
    assert row == [codes[0, 0] | codes[0, 2] << 4, codes[0, 4] | codes[0, 6] << 4, codes[0, 1] | codes[0, 3] << 4, codes[0, 5] | codes[0, 7] << 4]
    nan = torch.zeros(1, 32, dtype=BF)
    nan[0, 7] = math.inf
    assert U.values(*U.encode(nan)).isnan().all()
    big = torch.full((1, 32), 65504.0, dtype=HF)
    big[0, 1] = -65504.0
    assert torch.isfinite(U.values(*U.encode(big))).all()
    assert U.evict([5, 1, 1, 0, 3, 2], 4, 1, 1) == [0, 1, 4, 5] and U.evict([1.0, math.nan, 2.0], 1, 0, 0) == [1] and U.evict([1, 2], 2, 0, 0) == [0, 1]
    see = U.visible(3, 10, None, 4, 2)
    assert see[0].tolist() == [True] * 2 + [False] * 5 + [True] * 3 + [True, False, False]
    assert see[2].tolist() == [True] * 2 + [False] * 7 + [True] + [True] * 3
    assert U.visible(1, 3, None, 1, 0)[0].tolist() == [False, False, False, True]
    assert U.visible(6, 2, None, 3, 0)[5].tolist() == [False] * 2 + [False] * 3 + [True] * 3


def test_cache_refusals():
    u8 = torch.uint8
    for data, kw in ((_z(3, 2, 2, 640), {}), (_z(2, 2, 640, dtype=u8), {}), (_z(3, 2, 2, 600, dtype=u8), {}), (_z(3, 2, 0, 640, dtype=u8), {}),
                     (_z(3, 2, 2, 640, dtype=u8), dict(dtype=torch.float32)), (_z(3, 2, 640, 2, dtype=u8).transpose(2, 3), {}),
                     (_z(3, 2, 4, 640, dtype=u8)[:, :, ::2], {}), (_z(1, 2, 2, 640, dtype=u8).expand(3, 2, 2, 640), {}),
                     (_z(3, 1, 2, 640, dtype=u8).expand(3, 2, 2, 640), {}), (_z(1, 3, 2, 2, 640, dtype=u8).expand(2, 3, 2, 2, 640), {}),
                     (_z(3 * 2 * 1284 + 8, dtype=u8)[: 3 * 2 * 1284].view(3, 2, 1284)[..., :1280].view(3, 2, 2, 640), {})):
        with pytest.raises(ValueError, match="Int4Cache"):
            S.Int4Cache(data, **kw)
    for kw in (dict(page_size=12), dict(page_size=0), dict(dim=96), dict(pages=-1), dict(kv_heads=0)):
        with pytest.raises(ValueError, match="Int4Cache"):
            S.Int4Cache.empty(**{**dict(pages=2, page_size=16, kv_heads=1, dim=64, device="cpu"), **kw})
    with pytest.raises(ValueError, match="no layers"):
        _cache()[0]
    c = S.Int4Cache.empty(4, 24, 3, 128, HF, layers=2, device="cpu")
    assert (c.layers, c.pages, c.page_size, c.kv_heads, c.dim, c.dtype) == (2, 4, 24, 3, 128, HF) and c[1].layers is None
    assert c[1].data.data_ptr() == c.data.data_ptr() + 4 * 3 * 3 * 1280


def test_row_refusals():
    k, slots, i64 = _z(3, 2, 64, dtype=BF), _z(3, dtype=torch.int64), torch.int64
    c, l = _cache(), _cache(layers=2)
    for args, kw in (((k, k[:2], c, slots), {}), ((k.to(HF), k.to(HF), c, slots), {}), ((k, k.to(HF), c, slots), {}), ((k[:, :1], k[:, :1], c, slots), {}),
                     ((k, k, l, slots), {}), ((k[None], k[None], c, slots), {}), ((k[None], k[None], l, slots), {}), ((k, k, c, slots.int()), {}),
                     ((k, k, c, _z(4, dtype=i64)), {}), ((k, k, c, slots), dict(rows=_z(2))), ((k, k, c, slots), dict(rows=slots)),
                     ((_z(3, 2, 128, dtype=BF), _z(3, 2, 128, dtype=BF), c, slots), {})):
        with pytest.raises(ValueError, match="write_cache_int4"):
            S.write_cache_int4(*args, **kw)
    with pytest.raises(ValueError, match="read_cache_int4"):
        S.read_cache_int4(c, slots.int())


def _attention(**kw):
    return {**dict(q=_z(5, 4, 64, dtype=BF), k=_z(5, 2, 64, dtype=BF), v=_z(5, 2, 64, dtype=BF), cache=_cache(), tables=_z(2, 2), lengths=_z(2), starts=_z(3)), **kw}


def test_attention_refusals():
    f32 = torch.float32
    for kw in (dict(cache=_cache(layers=1)), dict(q=_z(5, 256, dtype=BF)), dict(k=_z(4, 2, 64, dtype=BF), v=_z(4, 2, 64, dtype=BF)), dict(v=_z(5, 1, 64, dtype=BF)),
               dict(q=_z(5, 4, 64, dtype=HF)), dict(q=_z(5, 4, 128, dtype=BF)), dict(cache=_cache(dtype=HF)), dict(cache=_cache(heads=1)), dict(cache=_cache(dim=128)),
               dict(tables=_z(2, 2, dtype=torch.int64)), dict(tables=_z(4)), dict(lengths=_z(3)), dict(lengths=_z(2, dtype=torch.int64)), dict(starts=_z(2)),
               dict(starts=_z(3, dtype=torch.int64)), dict(mask=_z(5)), dict(mask=_z(4, 1)), dict(mask=_z(5, 0)), dict(mask=_z(5, 1, dtype=torch.int64)),
               dict(out=_z(5, 4, 128, dtype=BF)[:, :, ::2]), dict(out=_z(5, 4, 64, dtype=HF)), dict(lse=_z(5, 2, dtype=f32)), dict(lse=_z(4, 5, dtype=f32).t()),
               dict(window=0), dict(window=-3), dict(sinks=4), dict(window=8, sinks=-1)):
        with pytest.raises(ValueError, match="tree_attention_int4"):
            S.tree_attention_int4(**_attention(**kw))


def _weights(**kw):
    return {**dict(q=_z(5, 4, 64, dtype=BF), cache=_cache(), tables=_z(2, 2), lengths=_z(2), starts=_z(3), lse=_z(5, 4, dtype=torch.float32),
                   weights=_z(2, 2, 40, dtype=torch.float32)), **kw}


def test_weights_refusals():
    f32 = torch.float32
    for kw in (dict(cache=_cache(layers=1)), dict(cache=_z(3, 16, 2, 64, dtype=f32)), dict(cache=_z(3, 12, 2, 64, dtype=BF)), dict(cache=_z(3, 16, 2, 96, dtype=BF)),
               dict(cache=_z(3, 16, 128, dtype=BF)), dict(cache=_z(3, 16, 64, 2, dtype=BF).transpose(2, 3)), dict(cache=_z(3, 16, 3, 64, dtype=BF)),
               dict(cache=_z(3, 16, 2, 68, dtype=BF)[..., :64]), dict(q=_z(5, 4, 64, dtype=HF)), dict(q=_z(5, 3, 64, dtype=BF)), dict(q=_z(20, 64, dtype=BF)),
               dict(q=_z(5, 4, 128, dtype=BF)), dict(tables=_z(4)), dict(lengths=_z(3)), dict(starts=_z(2)), dict(starts=_z(3, dtype=torch.int64)),
               dict(lse=_z(5, 2, dtype=f32)), dict(lse=_z(5, 4, dtype=BF)), dict(weights=_z(2, 1, 40, dtype=f32)), dict(weights=_z(2, 2, 40, dtype=BF)),
               dict(weights=_z(2, 40, 2, dtype=f32).transpose(1, 2)), dict(weights=_z(1, 2, 40, dtype=f32).expand(2, 2, 40)), dict(window=0),
               dict(sinks=1), dict(window=3, sinks=-2)):
        with pytest.raises(ValueError, match="attention_weights"):
            S.attention_weights(**_weights(**kw))


def _evict(**kw):
    return {**dict(cache=_cache(), tables=_z(2, 2), lengths=_z(2), weights=_z(2, 2, 40, dtype=torch.float32), keep=20), **kw}


def test_evict_refusals():
    f32 = torch.float32
    row = _z(3, 16, 2, 64, dtype=BF)
    for kw in (dict(cache=(row, row[:2])), dict(cache=(row, row.to(HF))), dict(cache=(row[0], row[0])), dict(cache=(row[:, :0], row[:, :0])),
               dict(cache=(row.transpose(2, 3), row.transpose(2, 3))), dict(cache=(_z(3, 16, 2, 68, dtype=BF)[..., :64],) * 2), dict(cache=(_z(3, 16, 2, 4, dtype=BF),) * 2),
               dict(cache=(row[:1].expand(3, 16, 2, 64), row)), dict(tables=_z(4)), dict(lengths=_z(3)), dict(weights=_z(2, 3, 40, dtype=f32)),
               dict(weights=_z(1, 2, 2, 40, dtype=f32)), dict(weights=_z(2, 2, 40, dtype=BF)), dict(cache=_cache(layers=2)),
               dict(cache=_cache(layers=2), weights=_z(1, 2, 2, 40, dtype=f32)), dict(keep=-1), dict(sinks=-1), dict(recent=-1), dict(sinks=15, recent=6)):
        with pytest.raises(ValueError, match="evict_cache"):
            S.evict_cache(**_evict(**kw))


def test_calls_have_no_cpu_form():
    k, slots = _z(3, 2, 64, dtype=BF), _z(3, dtype=torch.int64)
    for call in (lambda: S.write_cache_int4(k, k, _cache(), slots), lambda: S.read_cache_int4(_cache(), slots), lambda: S.tree_attention_int4(**_attention()),
                 lambda: S.attention_weights(**_weights()), lambda: S.attention_weights(**_weights(cache=_z(3, 16, 2, 64, dtype=BF))),
                 lambda: S.evict_cache(**_evict()), lambda: S.evict_cache(**_evict(cache=(_z(3, 16, 2, 64, dtype=BF),) * 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_tensors_on_other_devices_are_refused(monkeypatch):
    """Tensors that only claim to be on a device: no call gets as far as a pointer."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from actfold_b200.kernels import DeviceStatus

    cache = _cache()
    with FakeTensorMode():
        def z(*shape, dtype=torch.int32, on="cuda:1"):
            return torch.empty(*shape, dtype=dtype, device=on)

        cache.data = z(3, 2, 2, 640, dtype=torch.uint8)
        f32, i64 = torch.float32, torch.int64
        attention = dict(q=z(5, 4, 64, dtype=BF), k=z(5, 2, 64, dtype=BF), v=z(5, 2, 64, dtype=BF), cache=cache, tables=z(2, 2), lengths=z(2), starts=z(3))
        weights = dict(q=z(5, 4, 64, dtype=BF), cache=cache, tables=z(2, 2), lengths=z(2), starts=z(3), lse=z(5, 4, dtype=f32), weights=z(2, 2, 40, dtype=f32))
        evict = dict(cache=cache, tables=z(2, 2), lengths=z(2), weights=z(2, 2, 40, dtype=f32), keep=20)
        monkeypatch.setattr(K, "_row_strides", lambda t: (16, 16, 16))
        rows = dict(k=z(5, 2, 64, dtype=BF), v=z(5, 2, 64, dtype=BF), cache=cache, slots=z(5, dtype=i64))
        for fn, args in ((S.tree_attention_int4, attention), (S.attention_weights, weights), (S.evict_cache, evict), (S.write_cache_int4, rows),
                         (S.read_cache_int4, dict(cache=cache, slots=z(5, dtype=i64)))):
            for where, error in (("cuda:0", ValueError), ("cpu", RuntimeError)):
                with pytest.raises(error, match="cuda:0|CUDA device"):
                    fn(**args, status=DeviceStatus(where))
            for name, t in args.items():
                if isinstance(t, torch.Tensor):
                    with pytest.raises(ValueError, match="cuda:0"):
                        fn(**{**args, name: z(*t.shape, dtype=t.dtype, on="cuda:0")})


def _pack(struct, fields, **kw):
    return struct.pack(*(y for x in {**fields, **kw}.values() for y in (x if isinstance(x, tuple) else (x,))))


def test_entry_points_refuse_before_any_launch(lib):
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf)
    p += -p % 16
    cache = (p, 0, 2560, 1280, 1, 2, 16, 2, 64, 2)  # data, strides (layer, page, head), layers, pages, page_size, heads, head_dim, dtype
    bad_caches = [(0, *cache[1:]), (p + 8, *cache[1:]), (*cache[:2], 2568, *cache[3:]), (*cache[:6], 12, *cache[7:]), (*cache[:6], 0, *cache[7:]),
                  (*cache[:8], 80, 2), (*cache[:9], 0), (*cache[:9], 7), (*cache[:5], -1, *cache[6:]), (*cache[:5], 1 << 40, *cache[6:])]
    rows = dict(k=p, v=p, sk=(0, 256, 128), sv=(0, 256, 128), slots=p, rows=0, n=4, count=4, cache=cache)
    for call, name in ((lib.af_write_cache_int4, "write"), (lib.af_read_cache_int4, "read")):
        for kw in [dict(cache=c) for c in bad_caches] + [dict(k=0), dict(v=0), dict(slots=0), dict(count=-1), dict(sk=(0, 250, 128)), dict(k=p + 8), dict(count=1 << 40)]:
            assert call(_pack(K._ROWS, rows, **kw), None, None) == _lib.AF_ERR_ARG, (name, kw)
        assert call(None, None, None) == _lib.AF_ERR_ARG
        assert call(_pack(K._ROWS, rows, count=0), None, None) == _lib.AF_OK
    att = dict(q=p, k=p, v=p, sq=(512, 128), sk=(256, 128), sv=(256, 128), cache=cache, tables=p, ts=2, most=2, lengths=p, starts=p, mask=0, ms=0, words=0,
               batch=1, total=1, heads=4, window=0, sinks=0, scale=0.1, out=p, so=(512, 128), lse=0, ws=p, wsb=1 << 40)
    for kw in [dict(cache=c) for c in bad_caches] + [dict(q=0), dict(k=0), dict(out=0), dict(ws=0), dict(tables=0), dict(lengths=0), dict(heads=3), dict(heads=0),
                                                     dict(q=p + 8), dict(sk=(256, 130)), dict(batch=20000), dict(batch=-1), dict(mask=p), dict(mask=p, words=4, ms=3),
                                                     dict(mask=p, words=600, ms=600), dict(most=1 << 40), dict(wsb=0), dict(window=-1), dict(sinks=-1),
                                                     dict(total=1 << 27, heads=1 << 16), dict(total=1 << 28, most=1 << 20)]:
        assert lib.af_tree_attention_int4(_pack(K._ATTENTION, att, **kw), None, None) == _lib.AF_ERR_ARG, kw
    assert lib.af_tree_attention_int4(None, None, None) == _lib.AF_ERR_ARG
    assert lib.af_tree_attention_int4(_pack(K._ATTENTION, att, total=0), None, None) == _lib.AF_OK
    assert lib.af_tree_attention_int4(_pack(K._ATTENTION, att, batch=0), None, None) == _lib.AF_OK
    assert lib.af_tree_attention_int4_workspace_bytes(None) == _lib.AF_ERR_ARG
    wts = dict(q=p, sq=(512, 128), cache=cache, token=0, tables=p, ts=2, most=2, lengths=p, starts=p, batch=1, total=1, heads=4, window=0, sinks=0, scale=0.1,
               lse=p, weights=p, sw=(64, 32), places=32)
    for kw in [dict(cache=c) for c in bad_caches] + [dict(q=0), dict(lse=0), dict(weights=0), dict(tables=0), dict(heads=3), dict(sq=(512, 130)), dict(token=24),
                                                     dict(batch=-1), dict(window=-1), dict(sinks=-1), dict(places=-1), dict(most=1 << 40)]:
        assert lib.af_attention_weights(_pack(K._WEIGHTS, wts, **kw), None, None) == _lib.AF_ERR_ARG, kw
    assert lib.af_attention_weights(None, None, None) == _lib.AF_ERR_ARG
    for kw in (dict(total=0), dict(batch=0), dict(most=0)):
        assert lib.af_attention_weights(_pack(K._WEIGHTS, wts, **kw), None, None) == _lib.AF_OK
    none = (0,) * 10
    ev = dict(cache=cache, k=0, v=0, sk=(0,) * 4, sv=(0,) * 4, layers=0, pages=0, page=0, heads=0, hb=0, tables=p, ts=2, most=2, lengths=p, batch=1, weights=p,
              sw=(0, 64, 32), places=32, keep=20, sinks=2, recent=3, kept=p, wout=p, lout=p)
    rows16 = dict(cache=none, k=p, v=p, sk=(0, 4096, 256, 128), sv=(0, 4096, 256, 128), layers=1, pages=2, page=16, heads=2, hb=128)
    for kw in ([dict(cache=c) for c in bad_caches if c[9] == 2] + [{**rows16, **kw} for kw in (dict(k=0), dict(hb=24), dict(hb=8192), dict(page=0), dict(pages=-1), dict(sk=(0, 4096, 250, 128)))] +
               [dict(tables=0), dict(lengths=0), dict(weights=0), dict(kept=0), dict(wout=0), dict(lout=0), dict(keep=-1), dict(sinks=-1), dict(recent=19), dict(batch=-1),
                dict(places=-1), dict(most=1 << 40), dict(batch=1 << 30)]):
        assert lib.af_evict_cache(_pack(K._EVICT, ev, **kw), None, None) == _lib.AF_ERR_ARG, kw
    assert lib.af_evict_cache(None, None, None) == _lib.AF_ERR_ARG
    assert lib.af_evict_cache(_pack(K._EVICT, ev, batch=0), None, None) == _lib.AF_OK
