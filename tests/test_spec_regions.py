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
