"""The accepted rows' move (nwd_kv_commit), bit for bit, and the speculative step as a whole:
tree attention, verification and commit against token-by-token decoding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from devutil import bits, vals
from spec_ref import attention_bound, tree_attention, verify

pytestmark = pytest.mark.gpu
HD = 128


def _pools(rng, count, rows, nkv, hd=HD):
    return [rng.integers(0, 2 ** 16, (rows, nkv, hd), dtype=np.uint16) for _ in range(count)]


def _dev(pools):
    return [torch.from_numpy(p.view(np.float16).copy()).cuda() for p in pools]


def _commit(pools, off, pos, path, n):
    for p in pools:
        for b in range(len(off)):
            base = off[b] + pos[b]
            p[base:base + n[b]] = p[[base + x for x in path[b][:n[b]]]]


def _args(off, pos, path, n):
    i = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device="cuda")  # noqa: E731
    return i(off, torch.int64), i(pos), i(path), i(n)


@pytest.mark.parametrize("b,n,nkv,hd,count", [
    (1, 8, 8, 128, 8), (1, 1, 1, 128, 1), (5, 64, 8, 128, 2), (30, 17, 3, 128, 4), (3, 40, 2, 64, 16),
    (2, 33, 1, 8, 3), (70, 5, 4, 128, 18),
])
def test_commit_bit_exact(ops, b, n, nkv, hd, count):
    rng = np.random.default_rng(b + n)
    cap = 2 * n + 20
    pools = _pools(rng, count, b * cap, nkv, hd)
    off = [i * cap for i in range(b)]
    pos = [int(rng.integers(0, n + 20)) for _ in range(b)]
    acc = [int(rng.integers(0, n + 1)) for _ in range(b)]
    acc[0] = n if b > 1 else min(n, 5)
    path = [sorted(rng.choice(n, a, replace=False).tolist()) + [-1] * (n - a) for a in acc]
    dev = _dev(pools)
    sc = ops.Scratch()
    ops.kv_commit(dev, *_args(off, pos, path, acc), scratch=sc)
    _commit(pools, off, pos, path, acc)
    for d, p in zip(dev, pools):
        assert np.array_equal(bits(d), p)
    assert sc.check() == 0


def test_refused_paths_leave_the_rows(ops):
    rng = np.random.default_rng(1)
    n, cap = 6, 20
    path = [[0, 2, 1, 3, 4, 5], [0, 1, 6, -1, -1, -1], [-1, 0, 1, 2, 3, 4], [0, 0, 1, 2, 3, 4],
            [0, 2, 4, -1, -1, -1], [1, 3, 5, -1, -1, -1]]
    acc = [3, 3, 2, 2, 7, -1]
    pools = _pools(rng, 2, 6 * cap, 2)
    dev, sc = _dev(pools), ops.Scratch()
    ops.kv_commit(dev, *_args([i * cap for i in range(6)], [3] * 6, path, acc), scratch=sc)
    assert sc.check() == 4
    for d, p in zip(dev, pools):
        assert np.array_equal(bits(d), p)


def test_rows_outside_the_pool_are_refused(ops):
    rng = np.random.default_rng(2)
    pools = _pools(rng, 2, 40, 2)
    path, acc = [[0, 3, 4], [0, 2, -1], [1, 2, -1], [0, 1, 2]], [3, 2, 2, 3]
    for off, pos in (([0, 20, 10, -1], [36, 19, -11, 3]), ([2 ** 40, -30, 40, 39], [0, 2, 0, 0])):
        dev, sc = _dev(pools), ops.Scratch()
        ops.kv_commit(dev, *_args(off, pos, path, acc), scratch=sc)
        assert sc.check() == 2 | 4  # sequence 0's path also leaves its tree of 3 nodes
        for d, p in zip(dev, pools):
            assert np.array_equal(bits(d), p)
        wide, sc = [row + [-1, -1] for row in path], ops.Scratch()
        ops.kv_commit(dev, *_args(off, pos, wide, acc), scratch=sc)
        assert sc.check() == 2
        for d, p in zip(dev, pools):
            assert np.array_equal(bits(d), p)


def test_offsets_past_32_bits(ops):
    rows, nkv = 4_300_000, 8
    pool = torch.zeros(rows, nkv, HD, dtype=torch.float16, device="cuda")
    tail = torch.arange(1, 11, dtype=torch.float16, device="cuda")[:, None, None].expand(10, nkv, HD)
    pool[rows - 10:] = tail
    ops.kv_commit([pool], *_args([rows - 40], [30], [[0, 4, 9, -1, -1, -1, -1, -1, -1, -1]], [3]))
    want = torch.tensor([1., 5., 10., 4., 5., 6., 7., 8., 9., 10.], device="cuda")
    assert torch.equal(pool[rows - 10:, 3, 5].float(), want)
    assert not pool[:rows - 10].any()


def test_commit_in_a_graph_and_on_a_stream(ops):
    rng = np.random.default_rng(3)
    pools = _pools(rng, 4, 60, 8)
    args = _args([0, 30], [4, 9], [[0, 5, 6], [0, 7, 9]], [3, 3])
    path = torch.tensor([[0, 5, 6] + [-1] * 7, [0, 7, 9] + [-1] * 7], dtype=torch.int32, device="cuda")
    args = (args[0], args[1], path, args[3])
    s = torch.cuda.Stream()
    dev = _dev(pools)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ops.kv_commit(dev, *args)
    g.replay()
    torch.cuda.synchronize()
    other = _dev(pools)
    torch.cuda.synchronize()
    ops.kv_commit(other, *args, stream=s)
    s.synchronize()
    _commit(pools, [0, 30], [4, 9], path.tolist(), [3, 3])
    for a, d, p in zip(dev, other, pools):
        assert np.array_equal(bits(a), p) and np.array_equal(bits(d), p)


def test_speculative_steps_as_used(ops, engine_mod):
    """Three speculative steps of a small batch over two layers: every tree's outputs, every
    decision and every cache row against the 64-bit restatement, and a decode step at the end."""
    rng = np.random.default_rng(4)
    b, n, nh, nkv, vocab, ctx0 = 3, 11, 10, 2, 60, [33, 0, 120]
    layers = [engine_mod.BatchedDecodeAttention([200] * b, nh, nkv) for _ in range(2)]
    h = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    seqs = [[[h(c, nkv, HD), h(c, nkv, HD)] for c in ctx0] for _ in layers]
    for layer, rows in zip(layers, seqs):
        for i, c in enumerate(ctx0):
            layer.k_pool[i * 200:i * 200 + c] = t(rows[i][0])
            layer.v_pool[i * 200:i * 200 + c] = t(rows[i][1])
        layer.lengths.copy_(torch.tensor(ctx0, dtype=torch.int32))
    for _ in range(3):
        parents = np.stack([np.array([-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)],
                                     dtype=np.int32) for _ in range(b)])
        news = []
        for layer, rows in zip(layers, seqs):
            q, k, v = h(b, n, nh, HD), h(b, n, nkv, HD), h(b, n, nkv, HD)
            news.append((k, v))
            got = vals(layer.tree_step(t(q), t(k), t(v), t(parents)))
            for i in range(b):
                kk = np.concatenate([rows[i][0], k[i]]).astype(np.float64)
                vv = np.concatenate([rows[i][1], v[i]]).astype(np.float64)
                ref, mag, amp = tree_attention(q[i].astype(np.float64), kk, vv, len(rows[i][0]),
                                               parents[i], n, nkv, HD ** -0.5)
                assert (np.abs(got[i] - ref) <=
                        attention_bound(ref, mag, amp, len(kk), HD ** -0.5, 6.0)).all()
        z = rng.standard_normal((b, n, vocab)) * 2
        e = np.exp(z)
        target = (e / e.sum(-1, keepdims=True)).astype(np.float32)
        e = np.exp(z + rng.standard_normal(z.shape))
        draft = (e / e.sum(-1, keepdims=True)).astype(np.float32)
        tokens = rng.integers(0, vocab, (b, n), dtype=np.int32)
        u, w = rng.random((b, n), dtype=np.float32), rng.random(b, dtype=np.float32)
        path, count, token = ops.verify_tree(t(tokens), t(parents), t(target), t(u), t(w),
                                             draft_probs=t(draft))
        engine_mod.commit_layers(layers, path, count)
        for i in range(b):
            want, nxt = verify(tokens[i], parents[i], n, target[i], draft[i], u[i], w[i])
            assert path[i].tolist() == want + [-1] * (n - len(want)) and int(token[i]) == nxt
            for rows, (k, v) in zip(seqs, news):
                rows[i][0] = np.concatenate([rows[i][0], k[i][want]])
                rows[i][1] = np.concatenate([rows[i][1], v[i][want]])
    for layer, rows in zip(layers, seqs):
        assert layer.lengths.tolist() == [len(r[0]) for r in rows]
        assert layer.scratch.check() == 0
        for i in range(b):
            m = len(rows[i][0])
            assert np.array_equal(bits(layer.k_pool[i * 200:i * 200 + m]), rows[i][0].view(np.uint16))
            assert np.array_equal(bits(layer.v_pool[i * 200:i * 200 + m]), rows[i][1].view(np.uint16))
        q, k, v = h(b, nh, HD), h(b, nkv, HD), h(b, nkv, HD)
        got = vals(layer.step(t(q), t(k), t(v)))
        for i in range(b):
            kk = np.concatenate([rows[i][0], k[i][None]]).astype(np.float64)
            vv = np.concatenate([rows[i][1], v[i][None]]).astype(np.float64)
            ref, mag, amp = tree_attention(q[i][None].astype(np.float64), kk, vv, len(kk) - 1,
                                           np.array([-1]), 1, nkv, HD ** -0.5)
            assert (np.abs(got[i] - ref[0]) <=
                    attention_bound(ref, mag, amp, len(kk), HD ** -0.5, 6.0)[0]).all()


def test_layers_that_share_their_lengths(ops, engine_mod):
    layers = [engine_mod.BatchedDecodeAttention([20, 20], 4, 2) for _ in range(2)]
    layers[1].lengths = layers[0].lengths
    path = torch.tensor([[0, 2, -1], [0, -1, -1]], dtype=torch.int32, device="cuda")
    count = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    engine_mod.commit_layers(layers, path, count)
    assert layers[0].lengths.tolist() == [2, 1]
    with pytest.raises(ValueError, match="differ"):
        engine_mod.commit_layers([layers[0], layers[0]], path, count)


def test_tree_step_on_a_stream(ops, engine_mod):
    """A step on a stream that is not the current one, which still has work to do."""
    rng = np.random.default_rng(5)
    layer = engine_mod.BatchedDecodeAttention([64], 8, 2)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float16)).cuda()  # noqa: E731
    layer.k_pool.copy_(t(64, 2, HD))
    layer.v_pool.copy_(t(64, 2, HD))
    layer.lengths.fill_(20)
    q, k, v = t(1, 5, 8, HD), t(1, 5, 2, HD), t(1, 5, 2, HD)
    parents = torch.tensor([[-1, 0, 0, 1, 2]], dtype=torch.int32, device="cuda")
    want = layer.tree_step(q, k, v, parents).clone()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(10):
        trash = torch.mm(busy, busy)
        del trash
    got = layer.tree_step(q, k, v, parents, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
