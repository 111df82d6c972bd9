"""Speculative steps at the end of a sequence's region, and steps that are refused: the
neighbours' rows, the lengths and the layers' own places (engine.BatchedDecodeAttention)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from devutil import bits, vals
from spec_ref import attention_bound, random_parents, tree_attention

pytestmark = pytest.mark.gpu
HD = 128


def _t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _layer(engine_mod, rng, caps, lengths, nh=8, nkv=2):
    layer = engine_mod.BatchedDecodeAttention(caps, nh, nkv)
    layer.k_pool.copy_(_t(rng.standard_normal(layer.k_pool.shape).astype(np.float16)))
    layer.v_pool.copy_(_t(rng.standard_normal(layer.v_pool.shape).astype(np.float16)))
    layer.lengths.copy_(_i(lengths))
    return layer


def _trees(rng, b, n, nh=8, nkv=2):
    h = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    parents = np.stack([random_parents(rng, n) for _ in range(b)])
    return h(b, n, nh, HD), h(b, n, nkv, HD), h(b, n, nkv, HD), parents


def _check_output(got, q, k_rows, v_rows, ctx, parents, m, nkv):
    ref, mag, amp = tree_attention(q.astype(np.float64), k_rows.astype(np.float64),
                                   v_rows.astype(np.float64), ctx, parents, m, nkv, HD ** -0.5)
    tol = attention_bound(ref, mag, amp, len(k_rows), HD ** -0.5, 6.0)
    assert (np.abs(got - ref) <= tol).all()
    assert (got[m:] == 0).all()


@pytest.mark.parametrize("caps,lengths,n,tree_len", [
    ([40, 40, 40], [36, 10, 40], 6, None),
    ([40, 40, 40], [36, 10, 35], 6, [4, 6, 6]),     # the first one fits, the last does not
    ([100, 70, 300], [90, 69, 200], 61, [10, 2, 61]),
    ([64, 64, 64], [64, 0, 1], 64, None),
])
def test_a_tree_past_its_region_leaves_the_neighbour(ops, engine_mod, caps, lengths, n, tree_len):
    rng = np.random.default_rng(n)
    layer = _layer(engine_mod, rng, caps, lengths)
    q, k, v, parents = _trees(rng, len(caps), n)
    kp, vp = bits(layer.k_pool).copy(), bits(layer.v_pool).copy()
    got = vals(layer.tree_step(_t(q), _t(k), _t(v), _t(parents),
                               tree_len=None if tree_len is None else _i(tree_len)))
    assert layer.scratch.check() == 2
    off = np.cumsum([0] + caps)
    for b, ctx in enumerate(lengths):
        m = n if tree_len is None else tree_len[b]
        if ctx + m > caps[b]:
            assert (got[b] == 0).all()
            continue
        lo = off[b]
        kp[lo + ctx:lo + ctx + m] = k[b, :m].view(np.uint16)
        vp[lo + ctx:lo + ctx + m] = v[b, :m].view(np.uint16)
        f = lambda x: x[lo:lo + ctx + m].view(np.float16)  # noqa: E731
        _check_output(got[b], q[b], f(kp), f(vp), ctx, parents[b], m, 2)
    assert np.array_equal(bits(layer.k_pool), kp)
    assert np.array_equal(bits(layer.v_pool), vp)


def test_refused_trees_do_not_lengthen(ops, engine_mod):
    """A sequence whose tree the attention refused: rows and length stay, whatever was accepted."""
    rng = np.random.default_rng(3)
    caps, lengths, n = [30, 40, 50], [20, 35, 47], 5
    layers = [_layer(engine_mod, rng, caps, lengths) for _ in range(2)]
    q, k, v, parents = _trees(rng, 3, n)
    for layer in layers:
        layer.tree_step(_t(q), _t(k), _t(v), _t(parents))
    kp = [bits(p).copy() for layer in layers for p in (layer.k_pool, layer.v_pool)]
    path = [[0, 2, 4, -1, -1], [0, 1, 3, 4, -1], [0, -1, -1, -1, -1]]
    engine_mod.commit_layers(layers, _i(path), _i([3, 4, 1]))
    off = [0, 30, 70]
    for i, layer in enumerate(layers):
        assert layer.lengths.tolist() == [23, 39, 47]  # 47 + 5 > 50
        for j, pool in enumerate((layer.k_pool, layer.v_pool)):
            want = kp[2 * i + j]
            for b, m in ((0, 3), (1, 4)):
                base = off[b] + lengths[b]
                want[base:base + m] = want[[base + x for x in path[b][:m]]]
            assert np.array_equal(bits(pool), want)
    assert layers[0].scratch.check() == 2


def test_a_short_tree_in_a_region_without_room_for_the_longest(engine_mod):
    """What the attention takes the commit takes too: the tree's own length counts."""
    rng = np.random.default_rng(4)
    layer = _layer(engine_mod, rng, [30, 30], [26, 29])
    q, k, v, parents = _trees(rng, 2, 8)
    layer.tree_step(_t(q), _t(k), _t(v), _t(parents), tree_len=_i([4, 2]))
    layer.commit(_i([[0, 1, 3] + [-1] * 5, [0] + [-1] * 7]), _i([3, 1]))
    assert layer.lengths.tolist() == [29, 29]
    assert layer.scratch.check() == 2
    # the next step's trees are of another length
    layer.lengths.copy_(_i([10, 11]))
    layer.tree_step(_t(q), _t(k), _t(v), _t(parents))
    layer.commit(_i([[0, 5, 7] + [-1] * 5, [0, 6] + [-1] * 6]), _i([3, 2]))
    assert layer.lengths.tolist() == [13, 13]
    assert layer.scratch.check() == 0


@pytest.mark.parametrize("path,count", [
    ([0, 2, 1, 3, 4], 3), ([0, 0, 1, 2, 3], 2), ([-1, 0, 1, 2, 3], 2), ([0, 1, 5, -1, -1], 3),
    ([0, 1, 2, 3, 4], 6), ([0, 1, 2, 3, 4], -1), ([0, 4, -1, -1, -1], 2),  # node 4 is absent
])
def test_refused_paths_do_not_lengthen(engine_mod, path, count):
    rng = np.random.default_rng(5)
    layer = _layer(engine_mod, rng, [30, 30], [7, 9])
    q, k, v, parents = _trees(rng, 2, 5)
    layer.tree_step(_t(q), _t(k), _t(v), _t(parents), tree_len=_i([4, 5]))
    kp = bits(layer.k_pool).copy()
    layer.commit(_i([path, [0, 3, -1, -1, -1]]), _i([count, 2]))
    assert layer.lengths.tolist() == [7, 11]
    assert layer.scratch.check() == 4
    kp[30 + 9 + 1] = kp[30 + 9 + 3]
    assert np.array_equal(bits(layer.k_pool), kp)


@pytest.mark.parametrize("n_layers", [2, 3, 33])
def test_layers_keep_their_own_places(engine_mod, n_layers):
    """Layers of different lengths, and of different regions in pools of one size."""
    rng = np.random.default_rng(6)
    caps = [[20, 30], [30, 20], [25, 25]]
    lens = [[5, 9], [7, 3], [0, 19]]
    layers = [_layer(engine_mod, rng, caps[i % 3], lens[i % 3]) for i in range(n_layers)]
    path, count = [[0, 2, 5, -1, -1, -1], [0, 1, 3, 4, -1, -1]], [3, 4]
    before = [[bits(p).copy() for p in (layer.k_pool, layer.v_pool)] for layer in layers]
    engine_mod.commit_layers(layers, _i(path), _i(count))
    for i, (layer, pools) in enumerate(zip(layers, before)):
        off = [0, caps[i % 3][0]]
        for pool, want in zip((layer.k_pool, layer.v_pool), pools):
            for b in range(2):
                base = off[b] + lens[i % 3][b]
                want[base:base + count[b]] = want[[base + x for x in path[b][:count[b]]]]
            assert np.array_equal(bits(pool), want)
        assert layer.lengths.tolist() == [lens[i % 3][b] + count[b] for b in range(2)]
    assert layers[0].scratch.check() == 0


def test_a_sequence_that_one_layer_refuses_stays_in_all(engine_mod):
    rng = np.random.default_rng(7)
    layers = [_layer(engine_mod, rng, [20, 30], [5, 9]), _layer(engine_mod, rng, [20, 30], [18, 9])]
    before = [bits(p).copy() for layer in layers for p in (layer.k_pool, layer.v_pool)]
    engine_mod.commit_layers(layers, _i([[0, 2, -1], [0, 2, -1]]), _i([2, 2]))
    assert [layer.lengths.tolist() for layer in layers] == [[5, 11], [18, 11]]
    for pool, want in zip([p for layer in layers for p in (layer.k_pool, layer.v_pool)], before):
        want[20 + 9 + 1] = want[20 + 9 + 2]
        assert np.array_equal(bits(pool), want)
    assert layers[0].scratch.check() == 2


def test_steps_in_a_graph_up_to_the_end_of_the_region(engine_mod):
    """A captured step and commit, replayed until the trees no longer fit: the lengths stop."""
    rng = np.random.default_rng(8)
    layers = [_layer(engine_mod, rng, [24, 60], [3, 0]) for _ in range(2)]
    q, k, v, parents = (_t(x) for x in _trees(rng, 2, 6))
    path, count = _i([[0, 2, 3, -1, -1, -1], [0, 4, 5, -1, -1, -1]]), _i([3, 3])
    out = torch.empty_like(q)
    s = torch.cuda.Stream()

    def step():
        for layer in layers:
            layer.tree_step(q, k, v, parents, out=out)
        engine_mod.commit_layers(layers, path, count)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for _ in range(9):
        g.replay()
    torch.cuda.synchronize()
    for layer in layers:
        # 3 -> 21 in six steps of three (18 + 6 fit 24 rows, 21 + 6 do not); 0 -> 30 in ten
        assert layer.lengths.tolist() == [21, 30]
        kp = bits(layer.k_pool)
        src = bits(k)
        for at, b, nodes in ((0, 0, (0, 2, 3)), (24, 1, (0, 4, 5))):
            first = at + (3 if b == 0 else 0)
            for r in range(layer.lengths[b].item() - (3 if b == 0 else 0)):
                assert np.array_equal(kp[first + r], src[b, nodes[r % 3]])
    assert layers[0].scratch.check() == 2


@pytest.mark.parametrize("room,fits", [(37, True), (36, False), (0, False), (-5, False), (1000, True)])
@pytest.mark.parametrize("b", [1, 2])
def test_given_capacities(ops, b, room, fits):
    """The operator itself, in a pool that has room behind the sequence (both kernels)."""
    rng = np.random.default_rng(9)
    n, ctx, rows = 7, 30, 80
    q, k, v, parents = _trees(rng, b, n)
    pools = [_t(rng.standard_normal((rows, 2, HD)).astype(np.float16)) for _ in range(2)]
    old = [bits(p).copy() for p in pools]
    o = torch.full(q.shape, 9.0, dtype=torch.float16, device="cuda")
    sc = ops.Scratch()
    ops.kv_append_attention_tree(_t(q), _t(k), _t(v), *pools,
                                 torch.tensor([0, 40][:b], device="cuda"), _i([ctx] * b),
                                 _t(parents), o, 8, 2, capacity=_i([room] + [40] * (b - 1)),
                                 scratch=sc)
    got = vals(o)
    assert sc.check() == (0 if fits else 2)
    for x in range(b):
        if x == 0 and not fits:
            assert (got[0] == 0).all()
            continue
        lo = 40 * x + ctx
        old[0][lo:lo + n], old[1][lo:lo + n] = k[x].view(np.uint16), v[x].view(np.uint16)
        f = lambda a: a[40 * x:lo + n].view(np.float16)  # noqa: E731
        _check_output(got[x], q[x], f(old[0]), f(old[1]), ctx, parents[x], n, 2)
    assert np.array_equal(bits(pools[0]), old[0]) and np.array_equal(bits(pools[1]), old[1])
