"""Attention for a tree of drafted tokens (nwd_attn_tree, nwd_kv_append_attn_tree)
against the 64-bit restatement: node i attends the context, its ancestors and itself."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from devutil import bits, vals
from spec_ref import attention_bound, random_parents, tree_attention

pytestmark = pytest.mark.gpu
HD = 128


class Case:
    """Sequences with their regions in one pool, a guard of spare rows behind each."""

    def __init__(self, ctx, n, nh, nkv, seed, tree_len=None, chain=False, roots=False, guard=3):
        rng = np.random.default_rng(seed)
        self.ctx, self.n, self.nh, self.nkv = list(ctx), n, nh, nkv
        self.b = len(self.ctx)
        self.m = [n] * self.b if tree_len is None else list(tree_len)
        self.parents = np.stack([random_parents(rng, n, chain, roots) for _ in self.ctx])
        self.off = np.cumsum([0] + [c + n + guard for c in self.ctx])
        rows = int(self.off[-1])
        h = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
        self.k, self.v = h(rows, nkv, HD), h(rows, nkv, HD)
        self.q = h(self.b, n, nh, HD)
        self.tree_len = tree_len

    def dev(self):
        t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        return dict(q=t(self.q), k_pool=t(self.k), v_pool=t(self.v),
                    row_offset=t(self.off[:-1].astype(np.int64)),
                    seq_len=torch.tensor(self.ctx, dtype=torch.int32, device="cuda"),
                    parents=t(self.parents),
                    tree_len=None if self.tree_len is None else torch.tensor(
                        self.tree_len, dtype=torch.int32, device="cuda"))

    def check(self, o, scale=0.0, k=None, v=None, only=None):
        sc = scale or HD ** -0.5
        got = vals(o)
        assert got.shape == self.q.shape
        k, v = self.k if k is None else k, self.v if v is None else v
        for b in range(self.b) if only is None else only:
            lo, hi = self.off[b], self.off[b] + self.ctx[b] + self.m[b]
            kk, vv = k[lo:hi].astype(np.float64), v[lo:hi].astype(np.float64)
            ref, mag, amp = tree_attention(self.q[b].astype(np.float64), kk, vv, self.ctx[b],
                                           self.parents[b], self.m[b], self.nkv, sc)
            tol = attention_bound(ref, mag, amp, len(kk), sc, float(np.abs(vv).max(initial=0)))
            off = np.abs(got[b] - ref)
            assert np.isfinite(got[b]).all(), f"sequence {b}"
            assert (off <= tol).all(), f"sequence {b}: worst {np.max(off / tol):.2f} of the bound"
            assert (got[b, self.m[b]:] == 0).all(), f"sequence {b}: absent nodes"


def _attend(ops, d, nh, nkv, **kw):
    o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
    return ops.attention_tree(d["q"], d["k_pool"], d["v_pool"], d["row_offset"], d["seq_len"],
                              d["parents"], o, nh, nkv, HD, tree_len=d["tree_len"], **kw)


@pytest.mark.parametrize("ctx,n,nh,nkv", [
    ([150], 8, 40, 8),               # the engine's cache
    ([0], 1, 40, 8),                 # one token, no context: its own row
    ([0], 64, 8, 1),                 # no context, the largest tree, the largest group
    ([1], 3, 2, 2),                  # one row
    ([127], 1, 5, 1),                # a tree that ends with a 128-row block
    ([128], 1, 5, 1),                # ... and begins one
    ([100], 64, 40, 8),              # a tree across a block's end, several query tiles
    ([191], 64, 3, 3),               # group 1
    ([64, 0, 333, 127, 128, 129, 1000], 13, 14, 2),  # ragged, group 7
    ([300, 5], 33, 12, 4),           # group 3
    ([700, 20, 260], 43, 6, 2),      # 129 query rows: one past a tile
    ([5000], 5, 32, 8),              # long: split over the SMs
    ([4096, 30], 64, 40, 8),         # long and wide
    ([37] * 40, 4, 32, 8),           # many short sequences
    ([2000] * 9 + [0, 3], 9, 48, 8), # group 6
])
@pytest.mark.parametrize("chain", [False, True])
def test_tree_vs_f64(ops, ctx, n, nh, nkv, chain):
    c = Case(ctx, n, nh, nkv, seed=n * 7 + len(ctx), chain=chain)
    sc = ops.Scratch()
    c.check(_attend(ops, c.dev(), nh, nkv, scratch=sc))
    assert sc.check() == 0


def test_forest_and_scale(ops):
    """Several roots (each sees the context and its own line) and a given scale."""
    c = Case([77, 260], 21, 16, 4, seed=5, roots=True)
    c.check(_attend(ops, c.dev(), 16, 4, scale=0.31), scale=0.31)


@pytest.mark.parametrize("tree_len", [[0, 1, 17, 32, 5], [32, 31, 2, 0, 0]])
def test_tree_lengths(ops, tree_len):
    """Absent nodes: zero outputs, rows that are never read or written."""
    c = Case([130, 0, 511, 96, 250], 32, 20, 4, seed=6, tree_len=tree_len)
    d = c.dev()
    for b in range(c.b):  # what stands in the absent nodes' rows and the guard must not matter
        lo, hi = c.off[b] + c.ctx[b] + c.m[b], c.off[b + 1]
        d["k_pool"][lo:hi] = float("nan")
        d["v_pool"][lo:hi] = float("inf")
    c.check(_attend(ops, d, 20, 4))


def test_append_and_attend(ops):
    c = Case([150, 3, 1023, 0], 19, 40, 8, seed=7, tree_len=[19, 7, 18, 0])
    rng = np.random.default_rng(8)
    new = [rng.standard_normal((c.b, c.n, c.nkv, HD)).astype(np.float16) for _ in range(2)]
    d = c.dev()
    o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
    sc = ops.Scratch()
    ops.kv_append_attention_tree(d["q"], torch.from_numpy(new[0]).cuda(),
                                 torch.from_numpy(new[1]).cuda(), d["k_pool"], d["v_pool"],
                                 d["row_offset"], d["seq_len"], d["parents"], o, c.nh, c.nkv, HD,
                                 tree_len=d["tree_len"], scratch=sc)
    k, v = c.k.copy(), c.v.copy()
    for b in range(c.b):
        lo = c.off[b] + c.ctx[b]
        k[lo:lo + c.m[b]], v[lo:lo + c.m[b]] = new[0][b, :c.m[b]], new[1][b, :c.m[b]]
    assert np.array_equal(bits(d["k_pool"]), k.view(np.uint16))
    assert np.array_equal(bits(d["v_pool"]), v.view(np.uint16))
    c.check(o, k=k, v=v)
    assert sc.check() == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_rows_hold_anything(ops, bad):
    """A node's row with NaN or infinities reaches its descendants and nobody else."""
    c = Case([100, 128, 70], 30, 10, 2, seed=9)
    d = c.dev()
    victims = {0: 4, 1: 29, 2: 11}
    for b, j in victims.items():
        d["v_pool"][c.off[b] + c.ctx[b] + j] = bad
        d["k_pool"][c.off[b] + c.ctx[b] + j] = bad
    got = vals(_attend(ops, d, 10, 2))
    for b, j in victims.items():
        seers = []
        for i in range(c.n):
            up = i
            while up >= 0 and up != j:
                up = c.parents[b][up]
            if up == j:
                seers.append(i)
        rest = [i for i in range(c.n) if i not in seers]
        assert np.isfinite(got[b, rest]).all()
        assert np.isnan(got[b, seers]).all()  # an infinite or NaN score leaves no weights
        # those that do not see it come out as if the row held numbers
        ref, mag, amp = tree_attention(c.q[b].astype(np.float64),
                                       c.k[c.off[b]:c.off[b] + c.ctx[b] + c.n].astype(np.float64),
                                       c.v[c.off[b]:c.off[b] + c.ctx[b] + c.n].astype(np.float64),
                                       c.ctx[b], c.parents[b], c.n, c.nkv, HD ** -0.5)
        tol = attention_bound(ref, mag, amp, c.ctx[b] + c.n, HD ** -0.5, 6.0)
        assert (np.abs(got[b] - ref) <= tol)[rest].all()


@pytest.mark.parametrize("ctx", [40, 120])
def test_infinite_values_reach_only_descendants(ops, ctx):
    """V alone infinite in one column: descendants get it there, the other columns and the
    other nodes stay as they are."""
    c = Case([ctx], 12, 4, 2, seed=10, chain=False)
    d = c.dev()
    j, col = 3, 17
    d["v_pool"][ctx + j, :, col] = float("inf")
    d["v_pool"][ctx + j, :, col + 1] = -float("inf")
    got = vals(_attend(ops, d, 4, 2))
    ref, mag, amp = tree_attention(c.q[0].astype(np.float64), c.k[:ctx + 12].astype(np.float64),
                                   c.v[:ctx + 12].astype(np.float64), ctx, c.parents[0], 12, 2,
                                   HD ** -0.5)
    tol = attention_bound(ref, mag, amp, ctx + 12, HD ** -0.5, 6.0)
    sees = np.zeros(12, bool)
    for i in range(12):
        up = i
        while up >= 0:
            sees[i] |= up == j
            up = c.parents[0][up]
    assert sees.any() and not sees.all()
    assert (got[0, sees][..., col] == np.inf).all()
    assert (got[0, sees][..., col + 1] == -np.inf).all()
    keep = np.ones(HD, bool)
    keep[[col, col + 1]] = False
    near = np.abs(got[0] - np.where(np.isfinite(got[0]), ref, got[0])) <= tol
    assert near[~sees].all() and np.isfinite(got[0, ~sees]).all()
    assert near[sees][..., keep].all() and np.isfinite(got[0, sees][..., keep]).all()


def test_flat_tail_behind_one_large_score(ops):
    """Thousands of equal small weights behind one large one: none may be lost to rounding."""
    ctx, n = 16000, 2
    c = Case([ctx], n, 2, 1, seed=11, chain=True)
    c.q[:] = 0
    c.q[..., 0] = 8.0
    c.k[:] = 0
    c.k[5, :, 0] = 15.0                     # score 8 * 15 / sqrt(128) = 10.6 against 0
    c.v[:] = 0.5
    c.v[5] = -2.0
    c.check(_attend(ops, c.dev(), 2, 1))


def test_growing_scores(ops):
    """Every block's scores lie above the last one's: the running maximum moves each time."""
    ctx, n = 1500, 40
    c = Case([ctx], n, 8, 1, seed=12)
    c.q[..., 0] = 3.0
    c.k[:ctx + n, :, 0] = np.linspace(-60, 60, ctx + n)[:, None]
    c.check(_attend(ops, c.dev(), 8, 1))


def test_rows_outside_the_pool(ops):
    """Refused on the device: zero outputs, nothing written, the error word says which."""
    c = Case([90, 60, 70], 9, 8, 2, seed=13)
    for field, value in (("seq_len", 10 ** 6), ("seq_len", -1), ("row_offset", -5),
                         ("row_offset", 2 ** 40)):
        d = c.dev()
        d[field][1] = value
        sc = ops.Scratch()
        new = torch.ones(c.b, c.n, c.nkv, HD, dtype=torch.float16, device="cuda")
        o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
        ops.kv_append_attention_tree(d["q"], new, new, d["k_pool"], d["v_pool"], d["row_offset"],
                                     d["seq_len"], d["parents"], o, c.nh, c.nkv, HD, scratch=sc)
        assert sc.check() == 2
        assert (o[1] == 0).all()
        k, v = c.k.copy(), c.v.copy()
        for b in (0, 2):
            lo = c.off[b] + c.ctx[b]
            k[lo:lo + c.n], v[lo:lo + c.n] = 1, 1
        assert np.array_equal(bits(d["k_pool"]), k.view(np.uint16))
        assert np.array_equal(bits(d["v_pool"]), v.view(np.uint16))
        c.check(o, k=k, v=v, only=(0, 2))


def test_bad_parents_and_lengths(ops):
    """A parent at or past its node counts as -1, a length outside [0, N] as the nearer bound."""
    c = Case([50, 40, 30], 6, 8, 2, seed=14)
    d = c.dev()
    d["parents"][0] = torch.tensor([0, 0, 5, 2, -7, 2 ** 31 - 1], dtype=torch.int32)
    d["tree_len"] = torch.tensor([6, -3, 99], dtype=torch.int32, device="cuda")
    c.parents[0] = [-1, 0, -1, 2, -1, -1]
    c.m = [6, 0, 6]
    sc = ops.Scratch()
    c.check(_attend(ops, d, 8, 2, scratch=sc))
    assert sc.check() == 4


def test_chain_equals_decode_steps(ops, engine_mod):
    """A chain of nodes gives what as many decode steps give, within both kernels' bounds."""
    ctx, n = 400, 7
    c = Case([ctx], n, 40, 8, seed=15, chain=True, guard=0)
    d = c.dev()
    got = vals(_attend(ops, d, 40, 8))
    for i in range(n):
        o = torch.empty(40, HD, dtype=torch.float16, device="cuda")
        ops.attention(d["q"][0, i].contiguous(), d["k_pool"], d["v_pool"], o,
                      ops.AttnParams(40, 8, HD, ctx + i + 1))
        ref, mag, amp = tree_attention(c.q[0].astype(np.float64), c.k.astype(np.float64),
                                       c.v.astype(np.float64), ctx, c.parents[0], n, 8, HD ** -0.5)
        tol = attention_bound(ref, mag, amp, ctx + n, HD ** -0.5, 6.0)
        assert (np.abs(got[0, i] - vals(o)) <= 2 * tol[i]).all()


def test_repeated_calls_are_equal(ops):
    c = Case([3000, 17, 900], 24, 40, 8, seed=16)
    d = c.dev()
    first = _attend(ops, d, 40, 8).clone()
    for _ in range(5):
        assert torch.equal(_attend(ops, d, 40, 8), first)


def test_streams_and_graphs(ops):
    """Two graphs captured without a workspace of their own, replayed at the same time on
    two streams, and a call on a stream that is not the current one."""
    cs = [Case([5000, 12], 16, 32, 8, seed=17), Case([2500, 900], 16, 32, 8, seed=18)]
    ds = [c.dev() for c in cs]
    ref = [_attend(ops, d, 32, 8).clone() for d in ds]
    outs = [torch.zeros_like(r) for r in ref]
    streams = [torch.cuda.Stream() for _ in ds]
    graphs = []
    for d, o, s in zip(ds, outs, streams):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.attention_tree(d["q"], d["k_pool"], d["v_pool"], d["row_offset"], d["seq_len"],
                               d["parents"], o, 32, 8, HD)
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, r in zip(outs, ref):
        assert torch.equal(o, r)
    for handle in (streams[0], streams[0].cuda_stream):
        outs[0].zero_()
        torch.cuda.synchronize()
        ops.attention_tree(ds[0]["q"], ds[0]["k_pool"], ds[0]["v_pool"], ds[0]["row_offset"],
                           ds[0]["seq_len"], ds[0]["parents"], outs[0], 32, 8, HD, stream=handle)
        streams[0].synchronize()
        assert torch.equal(outs[0], ref[0])


def test_offsets_past_32_bits(ops):
    """Pool rows whose byte and element offsets pass 2^32."""
    nkv, n, ctx = 8, 10, 300
    rows = 4_300_000  # * 1024 halves = 4.4e9 elements
    k = torch.empty(rows, nkv, HD, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    c = Case([ctx, ctx], n, 16, nkv, seed=19, guard=0)
    d = c.dev()
    offs = [5, rows - ctx - n]
    for b, off in enumerate(offs):
        k[off:off + ctx + n] = d["k_pool"][c.off[b]:c.off[b + 1]]
        v[off:off + ctx + n] = d["v_pool"][c.off[b]:c.off[b + 1]]
    d["k_pool"], d["v_pool"] = k, v
    d["row_offset"] = torch.tensor(offs, dtype=torch.int64, device="cuda")
    c.check(_attend(ops, d, 16, nkv))


def test_given_workspace(ops):
    c = Case([700, 41], 12, 40, 8, seed=20)
    d = c.dev()
    ws = ops.TreeWorkspace(2, 12, 40, 8)
    ws._buf.fill_(255)  # whatever it held
    c.check(_attend(ops, d, 40, 8, workspace=ws))


@pytest.mark.parametrize("ctx,n,nh,nkv,tree_len", [
    ([300, 0, 1000, 64, 63, 2000, 5], 61, 40, 8, [61, 1, 25, 26, 0, 50, 51]),  # 25 nodes per tile
    ([700, 20, 90, 333, 128], 64, 8, 1, [17, 64, 0, 16, 48]),                  # 16 per tile, 4 tiles
    ([4000], 61, 40, 8, [25]), ([4000], 61, 40, 8, [26]), ([4000], 61, 40, 8, [61]),
    ([4000], 64, 16, 2, [33]), ([900], 64, 16, 2, [0]), ([0], 61, 40, 8, [7]),
    ([500] * 40, 60, 5, 1, [0] * 38 + [60, 1]),
])
def test_short_trees_of_several_tiles(ops, ctx, n, nh, nkv, tree_len):
    """Tiles without a present node: no work, zero outputs."""
    c = Case(ctx, n, nh, nkv, seed=sum(tree_len) + n, tree_len=tree_len)
    sc = ops.Scratch()
    c.check(_attend(ops, c.dev(), nh, nkv, scratch=sc))
    assert sc.check() == 0


@pytest.mark.parametrize("n,tree_len", [(2, None), (34, 3)])
def test_more_than_a_thousand_sequences(ops, n, tree_len):
    rng = np.random.default_rng(21)
    ctx = rng.integers(0, 90, 1100).tolist()
    lens = None if tree_len is None else rng.integers(0, tree_len + 1, 1100).tolist()
    if lens:
        lens[1050] = n
    c = Case(ctx, n, 4, 1, seed=22, tree_len=lens)
    c.check(_attend(ops, c.dev(), 4, 1))


def test_more_heads_than_processors(ops):
    c = Case([150], 3, 200, 200, seed=23)
    c.check(_attend(ops, c.dev(), 200, 200))


def test_output_aligned_to_16_bytes(ops):
    c = Case([90, 300], 11, 16, 4, seed=24)
    d = c.dev()
    buf = torch.full((c.q.size + 16,), 9.0, dtype=torch.float16, device="cuda")
    o = buf[8:-8].view(c.q.shape)
    assert o.data_ptr() % 32 == 16
    ops.attention_tree(d["q"], d["k_pool"], d["v_pool"], d["row_offset"], d["seq_len"],
                       d["parents"], o, 16, 4, HD)
    c.check(o)
    assert (buf[:8] == 9).all() and (buf[-8:] == 9).all()


@pytest.mark.parametrize("b", [1, 6])
@pytest.mark.parametrize("n", [5, 40])
def test_scores_that_keep_rising(ops, b, n):
    """Every block's largest score lies more than 2^8 above the block's before."""
    c = Case([700] * b, n, 16, 2, seed=25)
    c.q = np.abs(c.q)
    c.k = (np.sign(c.k) * 0.25).astype(np.float16)
    for i in range(b):
        c.k[c.off[i]:c.off[i] + 700] += (np.arange(700) // 64 * 1.5).astype(np.float16)[:, None, None]
    c.check(_attend(ops, c.dev(), 16, 2))


def test_nothing_to_do(ops):
    """No sequence, or no node: the output stays as it is."""
    k = torch.zeros(4, 2, HD, dtype=torch.float16, device="cuda")
    for b, n in ((0, 4), (2, 0)):
        q = torch.zeros(b, n, 8, HD, dtype=torch.float16, device="cuda")
        one = torch.zeros(b, dtype=torch.int32, device="cuda")
        par = torch.zeros(b, n, dtype=torch.int32, device="cuda")
        o = torch.empty_like(q)
        assert ops.attention_tree(q, k, k, one.long(), one, par, o, 8, 2) is o


def test_refusals_of_tensors(ops):
    c = Case([30, 50], 6, 8, 2, seed=26)
    d = c.dev()
    o = torch.empty_like(d["q"])

    def call(**kw):
        a = dict(d, o=o)
        ws = kw.pop("workspace", None)
        a.update(kw)
        ops.attention_tree(a["q"], a["k_pool"], a["v_pool"], a["row_offset"], a["seq_len"],
                           a["parents"], a["o"], 8, 2, HD, tree_len=a["tree_len"], workspace=ws)

    call()
    for kw in (dict(q=d["q"].float()), dict(row_offset=d["row_offset"].int()),
               dict(seq_len=d["seq_len"].long()), dict(parents=d["parents"].long()),
               dict(o=o.bfloat16()), dict(tree_len=d["seq_len"].float()), dict(q=None)):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(q=d["q"][:, :5].contiguous()), dict(q=d["q"].transpose(0, 1).contiguous()),
               dict(o=o.transpose(0, 1)), dict(seq_len=d["seq_len"][:1]),
               dict(k_pool=d["k_pool"][:-1]), dict(k_pool=d["k_pool"].transpose(0, 1)),
               dict(parents=d["parents"][0]), dict(q=d["q"].cpu()), dict(parents=d["parents"].cpu()),
               dict(q=torch.empty(2, 6, 8, 2 * HD, dtype=torch.float16, device="cuda")[..., ::2])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ops.NwdError):
        call(o=d["q"])
    small = ops.TreeWorkspace(2, 6, 8, 2)
    small.nbytes = 4096
    with pytest.raises(ops.NwdError):
        call(workspace=small)


# ---- one sequence in a small pool: csrc/tree_short.cu up to 2 048 rows and 64 query rows a head

@pytest.mark.parametrize("ctx,n,nh,nkv,tree_len", [
    (0, 1, 5, 1, None), (0, 8, 8, 1, None), (1, 64, 2, 2, None), (15, 1, 1, 1, None),
    (200, 8, 40, 8, None), (31, 16, 4, 1, [9]), (150, 8, 40, 8, [0]), (150, 8, 40, 8, [3]),
    (117, 8, 40, 8, None),   # a pool of 128 rows
    (118, 8, 40, 8, None),   # 129: a cluster
    (245, 8, 40, 8, None), (246, 8, 40, 8, None),
    (300, 1, 8, 1, None), (500, 33, 3, 3, None), (640, 12, 20, 4, [5]), (0, 12, 10, 2, None),
    (900, 64, 2, 2, None), (1500, 12, 40, 8, None), (2, 7, 8, 1, None),
    (2037, 8, 40, 8, None),  # 2 048
    (2038, 8, 40, 8, None),  # 2 049: the general kernel
    (150, 13, 40, 8, None),  # 65 query rows: the general kernel
])
@pytest.mark.parametrize("chain", [False, True])
def test_small_pool(ops, ctx, n, nh, nkv, tree_len, chain):
    guard = 260 if (ctx, n) in ((0, 12), (2, 7)) else 3  # few rows in many CTAs
    c = Case([ctx], n, nh, nkv, seed=ctx + n, tree_len=tree_len, chain=chain, guard=guard)
    d = c.dev()
    end = c.ctx[0] + c.m[0]
    d["k_pool"][end:] = float("nan")
    d["v_pool"][end:] = float("inf")
    sc = ops.Scratch()
    c.check(_attend(ops, d, nh, nkv, scratch=sc))
    assert sc.check() == 0


@pytest.mark.parametrize("ctx", [70, 1100])
@pytest.mark.parametrize("append", [False, True])
def test_small_pool_infinite_rows(ops, ctx, append):
    """Tree rows with NaN and infinities in V (and one in K) reach their descendants alone."""
    c = Case([ctx], 9, 10, 2, seed=31)
    v = c.v.copy()
    v[ctx + 3, 0, 5], v[ctx + 3, 1, 127] = np.inf, -np.inf
    v[ctx + 6, 1, 0], v[ctx + 6, 1, 64] = np.nan, 65504
    k = c.k.copy()
    k[ctx + 8] = np.nan
    d = c.dev()
    o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    if append:
        kp, vp = d["k_pool"].clone(), d["v_pool"].clone()
        kp[ctx:], vp[ctx:] = float("nan"), float("nan")
        ops.kv_append_attention_tree(d["q"], t(k[None, ctx:ctx + 9]), t(v[None, ctx:ctx + 9]), kp, vp,
                                     d["row_offset"], d["seq_len"], d["parents"], o, 10, 2)
        assert np.array_equal(bits(kp[:ctx + 9]), k[:ctx + 9].view(np.uint16))
        assert np.array_equal(bits(vp[:ctx + 9]), v[:ctx + 9].view(np.uint16))
    else:
        ops.attention_tree(d["q"], t(k), t(v), d["row_offset"], d["seq_len"], d["parents"], o, 10, 2)
    got = vals(o)[0]
    kk, vv = np.nan_to_num(k[:ctx + 9].astype(np.float64)), v[:ctx + 9].astype(np.float64)
    clean = np.where(np.isfinite(vv), vv, 0)
    ref, mag, amp = tree_attention(c.q[0].astype(np.float64), kk, clean, ctx, c.parents[0], 9, 2,
                                   HD ** -0.5)
    tol = attention_bound(ref, mag, amp, ctx + 9, HD ** -0.5, 65504.0)
    for i in range(9):
        line, j = [], i
        while j >= 0:
            line.append(j)
            j = int(c.parents[0, j])
        if 8 in line:
            assert np.isnan(got[i]).all()
            continue
        for h in range(10):
            extra = vv[[ctx + a for a in line], h // 5]
            extra = np.where(np.isfinite(extra), 0, extra).sum(0)
            ok = np.isfinite(extra)
            assert np.array_equal(got[i, h][~ok], extra[~ok], equal_nan=True)
            assert (np.abs(got[i, h] - ref[i, h])[ok] <= tol[i, h][ok]).all()


def test_small_pool_lengths_that_grow(ops):
    """One captured call, replayed as the sequence grows on the device."""
    for rows in (256, 700):
        c = Case([rows - 9], 6, 40, 8, seed=rows)
        d = c.dev()
        o = torch.zeros_like(d["q"])
        args = (d["q"], d["k_pool"], d["v_pool"], d["row_offset"], d["seq_len"], d["parents"], o, 40, 8)
        ops.attention_tree(*args)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.attention_tree(*args)
        for ctx in (0, 1, 17, 63, 64, 65, 128, 200, 247, rows - 9):
            d["seq_len"].fill_(ctx)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            c.ctx = [ctx]
            c.check(o)


def test_small_pool_rows_outside(ops):
    """A sequence that leaves the pool has no rows and no nodes."""
    for ctx in (100, 1000):
        c = Case([ctx], 6, 8, 2, seed=33, guard=0)
        d = c.dev()
        new = torch.ones(1, 6, 2, HD, dtype=torch.float16, device="cuda")
        for off, length in ((1, ctx), (-1, ctx), (0, ctx + 1), (0, -1), (2 ** 40, 3)):
            d["row_offset"].fill_(off)
            d["seq_len"].fill_(length)
            o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
            sc = ops.Scratch()
            ops.kv_append_attention_tree(d["q"], new, new, d["k_pool"], d["v_pool"], d["row_offset"],
                                         d["seq_len"], d["parents"], o, 8, 2, scratch=sc)
            assert (o == 0).all() and sc.check() != 0
        assert np.array_equal(bits(d["k_pool"]), c.k.view(np.uint16))
        assert np.array_equal(bits(d["v_pool"]), c.v.view(np.uint16))


@pytest.mark.parametrize("b", [1, 3])
def test_rows_outside_the_pool_with_several_tiles(ops, b):
    """All of such a sequence's nodes are absent, in every tile, without tree lengths too."""
    c = Case([900, 2000, 64][:b], 61, 40, 8, seed=40)
    d = c.dev()
    d["row_offset"][0] = c.off[-1] - 5
    sc = ops.Scratch()
    o = _attend(ops, d, 40, 8, scratch=sc)
    assert (o[0] == 0).all() and sc.check() == 2
    c.check(o, only=range(1, b))
