"""What the speculative-decoding calls refuse before any CUDA call (runs without a GPU)."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest
import torch


@pytest.fixture(scope="module")
def L(nwd):
    return import_module(nwd.__name__ + "._lib")


P = ctypes.c_void_p(256)
O = ctypes.c_void_p(512)  # an output apart from P  # noqa: E741


def _tree(lib, q=P, k=O, rows=100, off=P, parents=P, o=O, b=1, n=4, nh=8, nkv=2, hd=128, scale=0.0,
          ws=P, ws_bytes=1 << 40, new=None):
    f = ctypes.c_float(scale)
    if new is None:
        return lib.nwd_attn_tree(q, k, P, rows, off, P, parents, None, o, b, n, nh, nkv, hd, f, ws,
                                 ws_bytes, None, None)
    return lib.nwd_kv_append_attn_tree(q, new, P, k, P, rows, off, P, parents, None, o, b, n, nh,
                                       nkv, hd, f, ws, ws_bytes, None, None)


@pytest.mark.parametrize("new", [None, P])
def test_tree_attention_refusals(L, new):
    lib = L.load()
    odd = ctypes.c_void_p(264)
    for kw, status in [
        (dict(q=None), L.NWD_ERR_INVALID), (dict(k=None), L.NWD_ERR_INVALID),
        (dict(off=None), L.NWD_ERR_INVALID), (dict(parents=None), L.NWD_ERR_INVALID),
        (dict(o=None), L.NWD_ERR_INVALID), (dict(nh=0), L.NWD_ERR_INVALID),
        (dict(nkv=0), L.NWD_ERR_INVALID), (dict(nh=7), L.NWD_ERR_INVALID),
        (dict(hd=64), L.NWD_ERR_UNSUPPORTED), (dict(nh=18), L.NWD_ERR_UNSUPPORTED),
        (dict(n=65), L.NWD_ERR_UNSUPPORTED), (dict(b=4097), L.NWD_ERR_UNSUPPORTED),
        (dict(q=odd), L.NWD_ERR_INVALID), (dict(o=odd), L.NWD_ERR_INVALID),
        (dict(scale=-1.0), L.NWD_ERR_INVALID), (dict(scale=float("nan")), L.NWD_ERR_INVALID),
        (dict(scale=float("inf")), L.NWD_ERR_INVALID), (dict(rows=0), L.NWD_ERR_INVALID),
        (dict(rows=2 ** 31 + 1), L.NWD_ERR_INVALID),
        (dict(ws=None), L.NWD_ERR_WORKSPACE), (dict(ws=odd), L.NWD_ERR_WORKSPACE),
        (dict(ws_bytes=0), L.NWD_ERR_WORKSPACE), (dict(o=P), L.NWD_ERR_INVALID),
    ]:
        assert _tree(lib, new=new, **kw) == status, kw
        assert lib.nwd_last_error()
    assert _tree(lib, new=new, b=0) == L.NWD_OK
    assert _tree(lib, new=new, n=0) == L.NWD_OK
    if new is not None:
        assert _tree(lib, new=odd) == L.NWD_ERR_INVALID
        assert _tree(lib, new=new, k=P) == L.NWD_ERR_INVALID  # K and V in one pool


def test_workspace_size_refusals(L):
    lib, v = L.load(), ctypes.c_size_t()
    assert lib.nwd_attn_tree_workspace_size(1, 4, 8, 2, 128, None) == L.NWD_ERR_INVALID
    assert lib.nwd_attn_tree_workspace_size(1, 4, 8, 3, 128, ctypes.byref(v)) == L.NWD_ERR_INVALID
    assert lib.nwd_attn_tree_workspace_size(1, 65, 8, 2, 128, ctypes.byref(v)) == L.NWD_ERR_UNSUPPORTED
    assert lib.nwd_attn_tree_workspace_size(1, 4, 8, 2, 96, ctypes.byref(v)) == L.NWD_ERR_UNSUPPORTED


def test_verify_refusals(L):
    lib = L.load()

    def call(ptrs=None, b=1, n=4, vocab=100):
        a = [P, P, None, P, None, P, P, P, P, P]
        for i in ptrs or ():
            a[i] = None
        return lib.nwd_verify_tree(*a, b, n, vocab, None, None)

    for i in (0, 1, 3, 5, 6, 7, 8, 9):
        assert call(ptrs=[i]) == L.NWD_ERR_INVALID
    assert call(n=0) == L.NWD_ERR_INVALID
    assert call(vocab=0) == L.NWD_ERR_INVALID
    assert call(n=65) == L.NWD_ERR_UNSUPPORTED
    assert call(vocab=2 ** 31) == L.NWD_ERR_UNSUPPORTED
    assert call(b=65536) == L.NWD_ERR_UNSUPPORTED
    assert call(b=0) == L.NWD_OK


def test_commit_refusals(L):
    lib = L.load()

    def call(pools=(256, 512), off=P, pos=P, path=P, acc=P, b=1, n=4, nkv=2, hd=128):
        a = (ctypes.c_void_p * max(1, len(pools)))(*pools)
        return lib.nwd_kv_commit(a, len(pools), 100, off, pos, path, acc, b, n, nkv, hd, None, None)

    for kw in (dict(off=None), dict(pos=None), dict(path=None), dict(acc=None),
               dict(pools=(256, None)), dict(pools=(256, 256)), dict(nkv=0), dict(hd=0),
               dict(pools=tuple(256 * i for i in range(1, 18))), dict(nkv=1 << 20, hd=1 << 20)):
        assert call(**kw) == L.NWD_ERR_INVALID, kw
    for kw in (dict(pools=(264,)), dict(nkv=1, hd=4), dict(n=65), dict(b=65536)):
        assert call(**kw) == L.NWD_ERR_UNSUPPORTED, kw
    assert lib.nwd_kv_commit(None, 2, 100, P, P, P, P, 1, 4, 2, 128, None, None) == L.NWD_ERR_INVALID
    for kw in (dict(pools=()), dict(b=0), dict(n=0)):
        assert call(**kw) == L.NWD_OK, kw


def test_ops_refuse_cpu_tensors(ops):
    z = torch.zeros(1, 2, 8, 128, dtype=torch.float16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    one, off = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    pool = torch.zeros(10, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.attention_tree(z, pool, pool, off, one, i, z, 8, 2)
    f = torch.zeros(1, 2, 5)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.verify_tree(i, i, f, f[..., 0], f[:, 0, 0])
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.kv_commit([pool], off, one, i, one)
