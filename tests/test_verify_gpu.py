"""Verification of drafted tokens (nwd_verify_tree) against the 64-bit restatement: whole
numbers, equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from spec_ref import random_parents, verify

pytestmark = pytest.mark.gpu


def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _case(b, n, vocab, seed, near=1.0, sharp=2.0, chain=False, draft=True):
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((b, n, vocab)) * sharp
    target = _softmax(z)
    q = _softmax(z + near * rng.standard_normal(z.shape))
    parents = np.stack([random_parents(rng, n, chain) for _ in range(b)])
    tokens = np.zeros((b, n), np.int32)
    for i in range(b):
        for c in range(1, n):
            p = q[i, parents[i, c]].astype(np.float64)
            tokens[i, c] = rng.choice(vocab, p=p / p.sum()) if draft else \
                np.argsort(-p)[min(vocab - 1, c // 2)]
    u = rng.random((b, n), dtype=np.float32)
    w = rng.random(b, dtype=np.float32)
    return dict(tokens=tokens, parents=parents, target=target, draft=q if draft else None, u=u, w=w)


def _run(ops, c, tree_len=None, **kw):
    t = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    out = ops.verify_tree(t(c["tokens"]), t(c["parents"]), t(c["target"]), t(c["u"]), t(c["w"]),
                          draft_probs=t(c["draft"]),
                          tree_len=None if tree_len is None else torch.tensor(
                              tree_len, dtype=torch.int32, device="cuda"), **kw)
    return [x.cpu().numpy() for x in out]


def _check(ops, c, tree_len=None, parents=None, **kw):
    path, count, token = _run(ops, c, tree_len, **kw)
    b, n = c["tokens"].shape
    parents = c["parents"] if parents is None else parents
    for i in range(b):
        m = n if tree_len is None else min(max(tree_len[i], 0), n)
        want, nxt = verify(c["tokens"][i], parents[i], m, c["target"][i],
                           None if c["draft"] is None else c["draft"][i], c["u"][i], c["w"][i])
        assert list(path[i]) == want + [-1] * (n - len(want)), f"sequence {i}"
        assert count[i] == len(want) and token[i] == nxt, f"sequence {i}"
    return count


@pytest.mark.parametrize("b,n,vocab", [
    (1, 1, 50), (1, 2, 1), (3, 6, 7), (40, 12, 1000), (5, 64, 257), (2, 9, 131072), (7, 5, 50257),
    (130, 4, 4097), (300, 3, 33), (17, 8, 2047),
])
@pytest.mark.parametrize("draft", [True, False])
def test_verify_vs_f64(ops, b, n, vocab, draft):
    for chain in (False, True):
        c = _case(b, n, vocab, seed=b + n + vocab, chain=chain, draft=draft)
        sc = ops.Scratch()
        _check(ops, c, scratch=sc)
        assert sc.check() == 0


@pytest.mark.parametrize("draft", [True, False])
def test_every_child_rejected(ops, draft):
    """63 children of one node, all turned down: as many subtractions of the draft row."""
    c = _case(6, 64, 900, seed=3, near=2.0, draft=draft)
    c["parents"][:] = 0
    c["parents"][:, 0] = -1
    c["u"][:] = np.float32(1 - 2.0 ** -24)
    count = _check(ops, c)
    assert (count <= 2).all()


def test_identical_rows_accept_the_drawn_token(ops):
    """Where the draft is the target every drafted token stands, up to the last leaf."""
    c = _case(8, 7, 300, seed=4, chain=True)
    c["draft"] = c["target"].copy()
    rng = np.random.default_rng(5)
    for i in range(8):
        for k in range(1, 7):
            p = c["target"][i, k - 1].astype(np.float64)
            c["tokens"][i, k] = rng.choice(300, p=p / p.sum())
    c["u"][:] = np.float32(1 - 2.0 ** -24)
    assert (_check(ops, c) == 7).all()


def test_borders(ops):
    """Exact arithmetic in powers of two: u q = r is a rejection, a running sum that equals
    w sum(r) does not exceed it."""
    vocab = 8
    target = np.zeros((5, 3, vocab), np.float32)
    target[:, :] = np.array([1, 0, 2, 1, 0, 4, 0, 0], np.float32) / 8
    draft = np.full((5, 3, vocab), 0.125, np.float32)
    draft[:, :, 5], draft[:, :, 6] = 0.25, 0.0
    tokens = np.array([[0, 0, 0]] * 5, np.int32)
    tokens[:, 1] = [0, 0, 1, 5, 6]  # r = q: accepted for u < 1; r = 0; r = 2q; q = 0 and r = 0
    parents = np.array([[-1, 0, 0]] * 5, np.int32)
    u = np.zeros((5, 3), np.float32)
    u[:, 2] = 0.999
    u[1, 1] = np.float32(1 - 2.0 ** -24)
    w = np.array([0.125, 0.375, 0.5, 0.0, 0.499999], np.float32)
    c = dict(tokens=tokens, parents=parents, target=target, draft=draft, u=u, w=w)
    _check(ops, c)
    for x in (0.0, 0.125, 0.12499999, 0.375, 0.5, 0.9999999):
        c["w"][:] = x
        for draft_row in (draft, None):
            c["draft"] = draft_row
            _check(ops, c)


def test_nothing_left_of_the_row(ops):
    """Residuals without mass fall back to the whole row; a row without mass has no token."""
    vocab, n = 40, 4
    rng = np.random.default_rng(6)
    target = _softmax(rng.standard_normal((4, n, vocab)))
    draft = target.copy()
    target[1, 0] = 0
    target[2, 0] = 0
    target[2, 0, 7] = 1.0
    target[3, 0] = np.nan
    draft[0, 0, :] = 1.0  # covers the target: every rejection leaves nothing
    tokens = np.full((4, n), 7, np.int32)
    parents = np.array([[-1, 0, 0, 0]] * 4, np.int32)
    u = np.full((4, n), np.float32(1 - 2.0 ** -24))
    w = rng.random(4, dtype=np.float32)
    for d in (draft, None):
        c = dict(tokens=tokens, parents=parents, target=target, draft=d, u=u, w=w)
        _check(ops, c)
    _, _, token = _run(ops, c)
    assert token[1] == -1 and token[3] == -1


def test_nan_and_negative_entries_count_as_zero(ops):
    c = _case(9, 6, 500, seed=7)
    rng = np.random.default_rng(8)
    for name in ("target", "draft"):
        hit = rng.random(c[name].shape) < 0.1
        c[name][hit] = rng.choice(np.array([np.nan, -0.5, -np.inf, -0.0], np.float32), hit.sum())
    _check(ops, c)


@pytest.mark.parametrize("draft", [True, False])
def test_tree_lengths(ops, draft):
    c = _case(6, 20, 700, seed=9, draft=draft)
    _check(ops, c, tree_len=[20, 1, 0, 7, 19, 2])


def test_bad_tokens_parents_and_lengths(ops):
    c = _case(5, 8, 60, seed=10, near=0.1)
    c["tokens"][0, 1] = 60
    c["tokens"][1, 1:] = -1
    c["tokens"][2, 3] = 2 ** 31 - 1
    want = c["parents"].copy()
    c["parents"][3, 2] = 2
    c["parents"][3, 5] = 77
    c["parents"][4, 1] = -9
    want[3, 2] = want[3, 5] = want[4, 1] = -1
    sc = ops.Scratch()
    _check(ops, c, parents=want, scratch=sc)
    assert sc.check() == 4
    sc2 = ops.Scratch()
    c2 = _case(3, 8, 60, seed=11)
    _check(ops, c2, tree_len=[-1, 9, 8], scratch=sc2)
    assert sc2.check() == 4


def test_tokens_follow_the_target(ops):
    """What comes out is distributed as the target: the first token of 60 000 walks over a
    tree of two siblings and a grandchild, against 5 standard deviations of each count."""
    b, n, vocab = 60000, 4, 6
    rng = np.random.default_rng(12)
    p = np.array([0.30, 0.05, 0.25, 0.10, 0.20, 0.10], np.float32)
    q = np.array([0.10, 0.40, 0.10, 0.20, 0.05, 0.15], np.float32)
    target = np.broadcast_to(p, (b, n, vocab))
    draft = np.broadcast_to(q, (b, n, vocab))
    tokens = np.zeros((b, n), np.int32)
    tokens[:, 1:] = rng.choice(vocab, (b, n - 1), p=q.astype(np.float64) / q.astype(np.float64).sum())
    parents = np.array([[-1, 0, 0, 1]] * b, np.int32)
    points = tokens.copy()
    points[:, 1], points[:, 2] = 1, 4
    for d, t in ((draft, tokens), (None, points)):
        c = dict(tokens=t, parents=parents, target=target, draft=d,
                 u=rng.random((b, n), dtype=np.float32), w=rng.random(b, dtype=np.float32))
        path, count, token = _run(ops, c)
        first = np.where(count > 1, t[np.arange(b), np.maximum(path[:, 1], 0)], token)
        seen = np.bincount(first, minlength=vocab)
        pe = p.astype(np.float64) / p.astype(np.float64).sum()
        assert (np.abs(seen - b * pe) <= 5 * np.sqrt(b * pe * (1 - pe))).all(), seen


def test_unaligned_rows_stream_graph_and_out(ops):
    """Odd vocabularies put rows at every alignment; outputs in place, on a stream, replayed."""
    c = _case(11, 6, 1003, seed=13)
    t = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
    big = torch.empty(t["target"].numel() + 1, device="cuda")
    odd = big[1:].view(t["target"].shape)
    odd.copy_(t["target"])
    ref = ops.verify_tree(t["tokens"], t["parents"], t["target"], t["u"], t["w"],
                          draft_probs=t["draft"])
    out = tuple(torch.full_like(x, 77) for x in ref)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ops.verify_tree(t["tokens"], t["parents"], odd, t["u"], t["w"], draft_probs=t["draft"],
                          out=out, stream=s)
    s.synchronize()
    for a, r, o in zip(got, ref, out):
        assert a is o and torch.equal(a, r)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        res = ops.verify_tree(t["tokens"], t["parents"], odd, t["u"], t["w"],
                              draft_probs=t["draft"])
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for a, r in zip(res, ref):
        assert torch.equal(a, r)


def test_offsets_past_32_bits(ops):
    """A batch whose probabilities pass 2^32 elements: the last sequence's row is its own."""
    b, n, vocab = 200, 64, 340000
    target = torch.zeros(b, n, vocab, device="cuda")
    target[:, :, 11] = 1.0
    target[-1, -1, 11] = 0.0
    target[-1, -1, vocab - 1] = 1.0
    tokens = torch.full((b, n), 11, dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda").expand(b, n).contiguous()
    u = torch.full((b, n), 0.5, device="cuda")
    path, count, token = ops.verify_tree(tokens, parents, target, u, u[:, 0].contiguous())
    assert (count == n).all() and (token[:-1] == 11).all() and int(token[-1]) == vocab - 1
