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


NH, NKV, ROWS = 8, 2, 60
TREE = dict(q=B * N * NH * 256, k_new=B * N * NKV * 256, v_new=B * N * NKV * 256,
            k_pool=ROWS * NKV * 256, v_pool=ROWS * NKV * 256, row_offset=B * 8, seq_len=B * 4,
            capacity=B * 4, parents=B * N * 4, tree_len=B * 4, o=B * N * NH * 256)


def _tree(lib, p, append, err=None):
    v = {n: ctypes.c_void_p(x) for n, x in p.items()}
    tail = (v["o"], B, N, NH, NKV, 128, ctypes.c_float(0), ctypes.c_void_p(1 << 30), 1 << 40, err, None)
    if append:
        return lib.nwd_kv_append_attn_tree_bounded(
            v["q"], v["k_new"], v["v_new"], v["k_pool"], v["v_pool"], ROWS, v["row_offset"],
            v["seq_len"], v["capacity"], v["parents"], v["tree_len"], *tail)
    return lib.nwd_attn_tree(v["q"], v["k_pool"], v["v_pool"], ROWS, v["row_offset"], v["seq_len"],
                             v["parents"], v["tree_len"], *tail)


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("other", [n for n in TREE if n != "o"] + ["err"])
def test_tree_output(L, other, append):
    if other in ("k_new", "v_new", "capacity") and not append:
        return
    lib = L.load()
    for shift in (16 - TREE["o"], -256, 0, (TREE["o"] - 16 if other == "err" else
                                           (TREE[other] + 15) // 16 * 16 - 16)):
        p = {name: 1 << 20 | i << 17 for i, name in enumerate(TREE)}
        err = None
        if other == "err":
            err = ctypes.c_void_p(p["o"] + max(shift, 0))
        else:
            p["o"] = p[other] + shift
        assert _tree(lib, p, append, err) == L.NWD_ERR_INVALID, shift
        assert b"overlap" in lib.nwd_last_error()


def test_tree_pools(L):
    lib = L.load()
    for shift in (16 - TREE["k_pool"], TREE["k_pool"] - 16):
        p = {name: 1 << 20 | i << 17 for i, name in enumerate(TREE)}
        p["v_pool"] = p["k_pool"] + shift
        assert _tree(lib, p, True) == L.NWD_ERR_INVALID
        assert b"overlap" in lib.nwd_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("ctx", [20, 3000])
def test_tree_workspace(ops, ctx):
    """o beside the workspace, in one buffer, is served; o in its last bytes is refused."""
    import torch
    rows = ctx + N
    h = lambda *s: torch.randn(*s, device="cuda", dtype=torch.float16)  # noqa: E731
    q, k, v = h(1, N, NH, 128), h(rows, NKV, 128), h(rows, NKV, 128)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (torch.zeros(1, dtype=torch.int64, device="cuda"), i([ctx]), i([[-1, 0, 0, 1, 2]]))
    want = ops.attention_tree(q, k, v, *args, torch.empty_like(q), NH, NKV)
    ws = ops.TreeWorkspace(1, N, NH, NKV)
    buf = torch.zeros(ws.nbytes + q.numel() * 2, dtype=torch.uint8, device="cuda")
    ws._buf, ws.ptr = buf, buf.data_ptr()
    sc = ops.Scratch()
    for at, fits in ((ws.nbytes, True), (ws.nbytes - 256, False), (0, False)):
        o = buf[at:at + q.numel() * 2].view(torch.float16).view(q.shape)
        if not fits:
            with pytest.raises(ops.NwdError, match="overlap"):
                ops.attention_tree(q, k, v, *args, o, NH, NKV, workspace=ws)
            continue
        sc.ptr = ws.ptr  # the error word may be the workspace's first
        ops.attention_tree(q, k, v, *args, o, NH, NKV, workspace=ws, scratch=sc)
        assert torch.equal(o, want) and sc.check() == 0


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
