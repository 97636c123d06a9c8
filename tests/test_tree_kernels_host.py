"""Refusals of the tree verification operators, and their plain forms against hand-made answers (CPU only)."""

from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

import tree_util as U
from actfold_b200 import _lib
from actfold_b200 import speculative as S
from actfold_b200 import tree_kernels as T


def _z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from actfold_b200.build import build

        build()
    return _lib.load()


def test_plain_forms():
    assert U.ancestors([-1, 0, 0, 1, -1]) == [[0], [0, 1], [0, 2], [0, 1, 3], [4]]
    assert U.pack_bits([[0, 33]], 2).tolist() == [[1, 2]]
    # Tokens 7 -> 8 -> 9 agree, node 2 does not; the path is cut to two nodes.
    assert U.accept([-1, 0, 0, 1], [7, 8, 1, 9], [8, 9, 0, 5], 7, 4) == ([0, 1, 3], 5)
    assert U.accept([-1, 0, 0, 1], [7, 8, 1, 9], [8, 9, 0, 5], 7, 2) == ([0, 1], 9)
    assert U.accept([-1], [7], [3], 6, 2) == ([], 6) and U.accept([-1], [7], [3], None, 2) == ([0], 3)
    t, ring, slots, head, tail = U.tables_step([[4, 5, -1], [6, -1, -1]], [8, 4], [1, 4], [0, 3], [9, 8, 7], 3, 5, 4)
    assert t == [[4, 5, -1], [6, 9, -1]] and ring == [9, 8, 5] and slots == [[], [36, 37, 38]] and (head, tail) == (4, 6)


def test_wrappers_refuse_bad_shapes_and_types():
    i64 = torch.int64
    with pytest.raises(ValueError):
        S.tree_masks(_z(4, dtype=i64), _z(2), 1)
    with pytest.raises(ValueError):
        S.tree_masks(_z(4), _z(2), 0)
    with pytest.raises(ValueError):
        S.tree_masks(_z(4), _z(0), 1)
    with pytest.raises(ValueError):
        S.tree_masks(_z(4), _z(2), 1, _z(2))
    with pytest.raises(ValueError):
        S.accept_tree(_z(4), _z(4), _z(4, dtype=i64), _z(2), 3)
    with pytest.raises(ValueError):
        S.accept_tree(_z(4), _z(4, dtype=i64), _z(3, dtype=i64), _z(2), 3)
    with pytest.raises(ValueError):
        S.accept_tree(_z(4), _z(4, dtype=i64), _z(4, dtype=i64), _z(2), 0)
    with pytest.raises(ValueError):
        S.accept_tree(_z(4), _z(4, dtype=i64), _z(4, dtype=i64), _z(2), 2, _z(3, dtype=i64))
    tables = (_z(2, 3), _z(2), _z(2), _z(6), _z(2, dtype=i64))
    for bad in ((_z(2, 3, dtype=i64), *tables[1:]), (_z(3, 2).t(), *tables[1:]), (_z(1, 3).expand(2, 3), *tables[1:]),
                (tables[0], _z(3), *tables[2:]), (*tables[:3], _z(12)[::2], tables[4]), (*tables[:4], _z(2)), (*tables[:4], _z(3, dtype=i64))):
        with pytest.raises(ValueError):
            S.block_tables(*bad, 16, 8)
    for page, cap in ((0, 8), (16, -1)):
        with pytest.raises(ValueError):
            S.block_tables(*tables, page, cap)


def test_write_cache_refusals():
    h = torch.float16
    k, cache, slots = _z(3, 2, 64, dtype=h), _z(4, 8, 2, 64, dtype=h), _z(3, dtype=torch.int64)
    for args, kw in (((k, k[:2], cache, cache, slots), {}), ((k, k, cache, cache.float(), slots), {}), ((k, k, cache, cache, slots.int()), {}),
                     ((k, k, cache, cache, _z(4, dtype=torch.int64)), {}), ((k, k, cache, cache, slots), dict(rows=_z(2))),
                     ((k, k, cache, cache, slots), dict(rows=slots)), ((k, k, cache[:, :, :1], cache[:, :, :1], slots), {}),
                     ((k[None], k[None], cache, cache, slots), {}), ((k, k, cache.transpose(2, 3), cache.transpose(2, 3), slots), {}),
                     ((k, k, cache[:1].expand(4, 8, 2, 64), cache, slots), {}), ((k, k, cache[:, :0], cache[:, :0], slots), {})):
        with pytest.raises(ValueError):
            S.write_cache(*args, **kw)


def test_tree_attention_refusals():
    b = torch.bfloat16

    def case(**kw):
        a = dict(q=_z(5, 4, 64, dtype=b), k=_z(5, 2, 64, dtype=b), v=_z(5, 2, 64, dtype=b), k_cache=_z(3, 16, 2, 64, dtype=b),
                 v_cache=_z(3, 16, 2, 64, dtype=b), tables=_z(2, 2), lengths=_z(2), starts=_z(3))
        a.update(kw)
        return a

    for kw in (dict(q=_z(5, 256, dtype=b)), dict(k=_z(4, 2, 64, dtype=b), v=_z(4, 2, 64, dtype=b)), dict(v=_z(5, 1, 64, dtype=b)),
               dict(q=_z(5, 4, 64, dtype=torch.float16)), dict(q=_z(5, 4, 64, dtype=torch.float32)), dict(v_cache=_z(3, 16, 1, 64, dtype=b)),
               dict(k_cache=_z(3, 16, 1, 64, dtype=b), v_cache=_z(3, 16, 1, 64, dtype=b)), dict(tables=_z(2, 2, dtype=torch.int64)),
               dict(lengths=_z(3)), dict(starts=_z(2)), dict(mask=_z(5)), dict(mask=_z(4, 1)), dict(mask=_z(5, 1, dtype=torch.int64)),
               dict(out=_z(5, 4, 128, dtype=b)[:, :, ::2]), dict(out=_z(5, 4, 64, dtype=torch.float16)), dict(lse=_z(5, 2, dtype=torch.float32)),
               dict(k_cache=_z(3, 16, 2, 68, dtype=b)[..., :64]), dict(k_cache=_z(3, 16, 64, 2, dtype=b).transpose(2, 3))):
        with pytest.raises(ValueError):
            S.tree_attention(**case(**kw))


def test_wrappers_have_no_cpu_form():
    i64, b = torch.int64, torch.bfloat16
    with pytest.raises(RuntimeError, match="CUDA"):
        S.tree_masks(_z(4), _z(2), 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.accept_tree(_z(4), _z(4, dtype=i64), _z(4, dtype=i64), _z(2), 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.block_tables(_z(2, 3), _z(2), _z(2), _z(6), _z(2, dtype=i64), 16, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        S.write_cache(_z(3, 2, 64), _z(3, 2, 64), _z(4, 8, 2, 64), _z(4, 8, 2, 64), _z(3, dtype=i64))
    with pytest.raises(RuntimeError, match="CUDA"):
        S.tree_attention(_z(1, 2, 64, dtype=b), _z(1, 2, 64, dtype=b), _z(1, 2, 64, dtype=b), _z(3, 16, 2, 64, dtype=b),
                         _z(3, 16, 2, 64, dtype=b), _z(1, 2), _z(1), _z(2))


def test_branch_tree_packed():
    def node(name, parent, *tokens):
        return S.BranchNode(name, parent, torch.tensor([tokens]))

    tree = S.BranchTree(node("r", None, 7, 8))
    for n in (node("a", "r", 7, 8, 1), node("b", "r", 7, 8, 2), node("c", "a", 7, 8, 1, 3), node("d", "b", 7, 8, 2, 4), node("e", "a", 7, 8, 1, 5)):
        tree.add(n)
    ids, parents, tokens = tree.packed()
    assert ids == ["a", "b", "c", "e", "d"] and parents.tolist() == [-1, -1, 0, 0, 1] and tokens.tolist() == [1, 2, 3, 5, 4]
    assert parents.dtype is torch.int32 and tokens.dtype is torch.int64
    tree.prune("a")
    ids, parents, tokens = tree.packed()
    assert ids == ["b", "d"] and parents.tolist() == [-1, 0] and tokens.tolist() == [2, 4]
    assert U.accept(parents.tolist(), tokens.tolist(), [4, 9], 2, 8) == ([0, 1], 9)
    tree.add(node("f", "d", 7, 8, 2, 4, 1, 1))
    with pytest.raises(ValueError, match="one token"):
        tree.packed()
    empty = S.BranchTree(node("r", None, 7)).packed()
    assert empty[0] == [] and empty[1].numel() == 0 and empty[2].numel() == 0


def _attention_args(buf, **kw):
    p = C.addressof(buf)
    p += -p % 16
    a = dict(q=p, k=p, v=p, sq=(512, 128), sk=(256, 128), sv=(256, 128), kc=p, vc=p, skc=(4096, 256, 128), svc=(4096, 256, 128), pages=2, page=16,
             tables=p, ts=2, most=2, lengths=p, starts=p, mask=0, ms=0, words=0, batch=1, total=1, heads=4, kv=2, dim=64, dtype=2, scale=0.1,
             out=p, so=(512, 128), lse=0, ws=p, wsb=1 << 40)
    a.update(kw)
    return T._ATTENTION.pack(*(y for x in a.values() for y in (x if isinstance(x, tuple) else (x,))))


def test_entry_points_refuse_before_any_launch(lib):
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf)
    bad = [dict(q=0), dict(out=0), dict(kc=0), dict(ws=0), dict(dim=80), dict(dtype=0), dict(heads=3), dict(heads=130, kv=2), dict(page=12), dict(page=0),
           dict(q=p - p % 16 + 24), dict(sk=(256, 130)), dict(svc=(4096, 250, 128)), dict(batch=20000), dict(mask=p, words=0), dict(mask=p, words=4, ms=3),
           dict(mask=p, words=600, ms=600), dict(most=1 << 40), dict(wsb=0)]
    for kw in bad:
        if "q" in kw and kw["q"]:
            kw = dict(q=(p + -p % 16) + 8)
        assert lib.af_tree_attention(_attention_args(buf, **kw), None, None) in (_lib.AF_ERR_ARG, _lib.AF_ERR_CAPACITY), kw
    assert lib.af_tree_attention(None, None, None) == _lib.AF_ERR_ARG
    assert lib.af_tree_attention(_attention_args(buf, total=0), None, None) == _lib.AF_OK  # nothing to do
    assert lib.af_tree_attention_workspace_bytes(None) == _lib.AF_ERR_ARG
    assert lib.af_tree_masks(p, p, 1, 4, 0, None, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_tree_masks(p, p, 1, 4, 600, None, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_tree_masks(None, p, 1, 4, 1, None, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_tree_masks(p, p, 70000, 4, 1, None, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_accept_tree(p, p, p, p, 1, 4, 4, None, 0, p, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_accept_tree(p, p, p, p, 1, 4, 20000, None, 3, p, p, p, None, None) == _lib.AF_ERR_ARG
    assert lib.af_accept_tree(None, p, p, p, 1, 4, 4, None, 3, p, p, p, None, None) == _lib.AF_ERR_ARG
    ok = [p, 4, 4, None, p, p, 1, p, 8, p, 16, 8, 0, p, p, p, p + 64, None, None]
    for at, x in ((6, 0), (6, 20000), (8, 0), (10, 0), (11, -1), (12, 3), (4, None), (7, None), (16, p)):
        args = list(ok)
        args[at] = x
        assert lib.af_block_tables(*args) == _lib.AF_ERR_ARG, (at, x)
    rows = dict(k=p, v=p, sk=(0, 0, 0), sv=(0, 0, 0), kc=p, vc=p, skc=(0, 0, 0, 0), svc=(0, 0, 0, 0), slots=p, rows=0, n=1, count=1, pages=1, page=16,
                layers=1, heads=1, hb=16)

    def packed(**kw):
        return T._ROWS.pack(*(y for x in {**rows, **kw}.values() for y in (x if isinstance(x, tuple) else (x,))))

    for kw in (dict(k=0), dict(vc=0), dict(slots=0), dict(page=0), dict(count=-1), dict(hb=1 << 24), dict(heads=1 << 24)):
        assert lib.af_write_cache(packed(**kw), None, None) == _lib.AF_ERR_ARG, kw
    assert lib.af_write_cache(None, None, None) == _lib.AF_ERR_ARG
    assert lib.af_write_cache(packed(count=0), None, None) == _lib.AF_OK


def test_wait_limit_refusals(lib):
    for attempts in (-2, (1 << 18) + 1, 1 << 40):
        assert lib.af_tree_attention_wait_limit(attempts) == _lib.AF_ERR_ARG
    for attempts in (0, 1 << 18, -1):
        assert lib.af_tree_attention_wait_limit(attempts) == _lib.AF_OK


def test_a_status_on_another_device_is_refused(monkeypatch):
    """Tensors that only claim to be on a device: no call gets as far as a pointer."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from actfold_b200.kernels import DeviceStatus

    monkeypatch.setattr(T, "_cache_grid", lambda t: (16, 16, 16))
    i64, b = torch.int64, torch.bfloat16
    with FakeTensorMode():
        def z(*shape, dtype=torch.int32):
            return torch.empty(*shape, dtype=dtype, device="cuda:1")

        rows, cache = z(5, 2, 64, dtype=b), z(3, 16, 2, 64, dtype=b)
        for where, error in (("cuda:0", ValueError), ("cpu", RuntimeError)):
            st = DeviceStatus(where)
            for call in (lambda: S.tree_masks(z(4), z(2), 1, status=st),
                         lambda: S.accept_tree(z(4), z(4, dtype=i64), z(4, dtype=i64), z(2), 3, status=st),
                         lambda: S.block_tables(z(2, 3), z(2), z(2), z(6), z(2, dtype=i64), 16, 4, status=st),
                         lambda: S.write_cache(rows, rows, cache, cache, z(5, dtype=i64), status=st),
                         lambda: S.tree_attention(rows, rows, rows, cache, cache, z(2, 2), z(2), z(3), status=st)):
                with pytest.raises(error, match="cuda:0|CUDA device"):
                    call()


def test_host_classes_import_where_torch_has_no_cuda_names():
    """A torch without CUDA has neither name; the trees and policies of a host need none of them."""
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    delattr(torch._C, name)\n"
            "from actfold_b200.speculative import BranchNode, BranchTree, GreedyAcceptancePolicy\n"
            "GreedyAcceptancePolicy()\n"
            "assert BranchTree(BranchNode('r', None, torch.tensor([[1]]))).packed()[0] == []\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr
