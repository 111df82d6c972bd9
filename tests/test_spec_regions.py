"""What the speculative calls over sequences' own regions refuse (runs without a GPU)."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest


@pytest.fixture(scope="module")
def L(nwd):
    return import_module(nwd.__name__ + "._lib")


P = ctypes.c_void_p(256)
Q = ctypes.c_void_p(512)


def test_commit_layers_refusals(L):
    lib = L.load()

    def call(pools=(256, 512, 768, 1024), n_layers=None, off=(256, 256), pos=(256, 256), cap=None,
             tree=None, path=P, acc=P, b=1, n=4, nkv=2, hd=128):
        arr = lambda x: None if x is None else (ctypes.c_void_p * max(1, len(x)))(*x)  # noqa: E731
        layers = len(pools) // 2 if n_layers is None else n_layers
        return lib.nwd_kv_commit_layers(arr(pools), layers, 100, arr(off), arr(pos), arr(cap),
                                        arr(tree), path, acc, b, n, nkv, hd, None, None)

    for kw in (dict(off=None), dict(pos=None), dict(path=None), dict(acc=None), dict(pools=None, n_layers=2),
               dict(off=(256, None)), dict(pos=(None, 256)), dict(pools=(256, 512, None, 768)),
               dict(pools=(256, 512, 768, 256)), dict(n_layers=33), dict(nkv=0), dict(hd=0),
               dict(nkv=1 << 20, hd=1 << 20)):
        assert call(**kw) == L.NWD_ERR_INVALID, kw
        assert lib.nwd_last_error()
    for kw in (dict(pools=(256, 264, 512, 768)), dict(nkv=1, hd=4), dict(n=65), dict(b=65536)):
        assert call(**kw) == L.NWD_ERR_UNSUPPORTED, kw
    for kw in (dict(pools=(), off=None, pos=None), dict(b=0), dict(n=0),
               dict(b=0, cap=(256, None), tree=(None, 256))):
        assert call(**kw) == L.NWD_OK, kw


def test_bounded_append_refusals(L):
    lib = L.load()

    def call(q=P, new=P, k=Q, cap=P, o=Q, b=1, n=4, nh=8, ws=P, ws_bytes=1 << 40):
        return lib.nwd_kv_append_attn_tree_bounded(q, new, P, k, P, 100, P, P, cap, P, None, o, b,
                                                   n, nh, 2, 128, ctypes.c_float(0), ws, ws_bytes,
                                                   None, None)

    for cap in (P, None):
        for kw, status in [(dict(q=None), L.NWD_ERR_INVALID), (dict(new=None), L.NWD_ERR_INVALID),
                           (dict(o=P), L.NWD_ERR_INVALID), (dict(k=P), L.NWD_ERR_INVALID),
                           (dict(n=65), L.NWD_ERR_UNSUPPORTED), (dict(nh=7), L.NWD_ERR_INVALID),
                           (dict(ws=None), L.NWD_ERR_WORKSPACE),
                           (dict(ws_bytes=0), L.NWD_ERR_WORKSPACE)]:
            assert call(cap=cap, **kw) == status, kw
        assert call(cap=cap, b=0) == L.NWD_OK and call(cap=cap, n=0) == L.NWD_OK
