"""Outputs that share memory with what the kernels still read are refused (runs without a GPU:
every call here is refused before any CUDA call)."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest

B, N, V = 3, 5, 40
# what a call of this size has in memory, in bytes, and where it lies if nothing overlaps
VERIFY = dict(tokens=B * N * 4, parents=B * N * 4, tree_len=B * 4, target=B * N * V * 4,
              draft=B * N * V * 4, u=B * N * 4, w=B * 4, path=B * N * 4, n_accepted=B * 4,
              next_token=B * 4)
OUT = ("path", "n_accepted", "next_token")


@pytest.fixture(scope="module")
def L(nwd):
    return import_module(nwd.__name__ + "._lib")


def _places(sizes):
    return {name: 1 << 20 | i << 14 for i, name in enumerate(sizes)}


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("other", [n for n in VERIFY])
def test_verify_outputs(L, out, other):
    if out == other:
        return
    lib = L.load()
    for at in ("same", "first byte", "last byte"):
        p = _places(VERIFY)
        p[out] = {"same": p[other], "first byte": p[other] - VERIFY[out] + 4,
                  "last byte": p[other] + VERIFY[other] - 4}[at]
        args = [ctypes.c_void_p(p[n]) for n in VERIFY]
        assert lib.nwd_verify_tree(*args, B, N, V, None, None) == L.NWD_ERR_INVALID, at
        assert b"overlap" in lib.nwd_last_error()


@pytest.mark.parametrize("out", OUT)
def test_verify_error_word(L, out):
    lib, p = L.load(), _places(VERIFY)
    args = [ctypes.c_void_p(p[n]) for n in VERIFY]
    assert lib.nwd_verify_tree(*args, B, N, V, ctypes.c_void_p(p[out] + 4), None) == L.NWD_ERR_INVALID
    assert b"overlap" in lib.nwd_last_error()


@pytest.mark.gpu
def test_outputs_side_by_side(ops):
    """Neighbours in one buffer do not overlap; the tokens' own memory as path is refused."""
    import torch
    target = torch.softmax(torch.randn(B, N, V, device="cuda"), -1)
    buf = torch.full((B * N * 3 + 2 * B + 2,), 7, dtype=torch.int32, device="cuda")
    tokens, parents, path = (buf[1 + i * B * N:1 + (i + 1) * B * N].view(B, N) for i in range(3))
    tokens.zero_()
    parents.copy_(torch.arange(-1, N - 1, dtype=torch.int32))
    count, token = buf[1 + 3 * B * N:][:B], buf[1 + 3 * B * N + B:][:B]
    u, w = torch.full((B, N), 0.999, device="cuda"), torch.full((B,), 0.5, device="cuda")
    want = ops.verify_tree(tokens, parents, target, u, w)
    ops.verify_tree(tokens, parents, target, u, w, out=(path, count, token))
    for a, b in zip((path, count, token), want):
        assert torch.equal(a, b)
    assert buf[0] == 7 and buf[-1] == 7
    with pytest.raises(ops.NwdError, match="overlap"):
        ops.verify_tree(tokens, parents, target, u, w, out=(tokens, count, token))
