"""CPU models of the tree-attention kernel's work split and of its turn protocol
(csrc/tree_attn.cu), which cannot be looked into on the GPU.

* the split: the CTAs' pieces cover every unit's blocks once, every unit that a cut divides
  has exactly one joining CTA, whose piece list is the unit's, and no partial slot is used twice;
* the protocol: the MMA issuers, producers and the two softmax groups, with mbarriers that only
  know the parity of their phase, run under random timing to the end, each turn's softmax
  reads the scores of its own block, and no accumulator or stage is overwritten in use.
"""
from __future__ import annotations

import random

import pytest

BN = 64


def pieces(blocks, n_units, ctas, min_blocks=1):
    """Per CTA the list of (b, u, blk, nb), and the joins (cta -> (b, u, first))."""
    line = [(b, u, n) for b, n in enumerate(blocks) for u in range(n_units)]
    total = sum(n for _, _, n in line)
    per = max(-(-total // ctas), min_blocks)
    out, joins = [], {}
    for c in range(ctas):
        x0, x1 = min(total, c * per), min(total, c * per + per)
        mine, at = [], 0
        for b, u, n in line:
            lo, hi = max(x0, at), min(x1, at + n)
            if lo < hi:
                mine.append((b, u, lo - at, hi - lo))
                if lo > at and hi == at + n:
                    joins[c] = (b, u, at // per)
            at += n
        out.append(mine)
    return out, joins


@pytest.mark.parametrize("seed", range(12))
def test_split_covers_every_unit(seed):
    r = random.Random(seed)
    blocks = [r.choice([1, 1, 2, 5, 33, r.randint(1, 400)]) for _ in range(r.choice([1, 2, 7, 64]))]
    n_units, ctas = r.choice([1, 2, 8, 16]), r.choice([1, 7, 148])
    got, joins = pieces(blocks, n_units, ctas, r.choice([1, 3]))
    seen, slots = {}, set()
    for c, mine in enumerate(got):
        for b, u, blk, nb in mine:
            seen.setdefault((b, u), []).append((blk, nb, c))
            if not (blk == 0 and nb == blocks[b]):
                slot = (c, 0 if blk > 0 else 1)
                assert slot not in slots
                slots.add(slot)
    for (b, u), parts in seen.items():
        at = 0
        for blk, nb, _ in parts:
            assert blk == at
            at += nb
        assert at == blocks[b]
        joining = [c for c, (jb, ju, _) in joins.items() if (jb, ju) == (b, u)]
        if len(parts) == 1:
            assert not joining
        else:
            assert joining == [parts[-1][2]]
            first = joins[joining[0]][2]
            cs = [c for _, _, c in parts]
            assert cs == list(range(first, joining[0] + 1))
            assert parts[0][0] == 0 and all(blk > 0 for blk, _, _ in parts[1:])
    assert len(seen) == len(blocks) * n_units


class Bar:
    """An mbarrier: a wait for a parity passes when the phase before the current one has it."""

    def __init__(self, count):
        self.count, self.left, self.done = count, count, 0

    def arrive(self, n=1):
        assert self.left >= n
        self.left -= n
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1

    def passed(self, parity):
        return (self.done - 1) & 1 == parity


def protocol(plan, seed, NQ=2, NK=5, NV=5, in_order=True):
    """plan: [(nb, tiles)] per piece.  Roles are generators that yield until a wait passes."""
    rnd = random.Random(seed)
    bars = {}

    def bar(name, i, count=1):
        return bars.setdefault((name, i), Bar(count))

    for name, n in (("QE", NQ), ("KE", NK), ("VE", NV)):
        for i in range(n):
            bar(name, i, 2)
    for g in range(2):
        bar("P", 2 * g, 2), bar("P", 2 * g + 1, 2), bar("OE", g, 4), bar("ML", g, 2)  # two threads stand for a group's 128
    q, k, v = [None] * NQ, [None] * NK, [None] * NV
    s_buf, o_buf, log = [None] * 4, [None, None], []
    mmas = [[], [], [], []]  # issued by an issuer, not yet run, in order

    def wait(b, parity):
        while not b.passed(parity):
            yield

    flying = []  # copies land in any order

    def copy(store, i, item, full):
        store[i] = None
        flying.append((store, i, item, full))

    def copies():
        while True:
            if flying and rnd.random() < 0.3:
                store, i, item, full = flying.pop(rnd.randrange(len(flying)))
                store[i] = item
                full.arrive()
            yield

    def load(kind, slots, store, items):
        i, ph = 0, 0
        for item in items:
            yield from wait(bar(kind + "E", i), ph ^ 1)
            copy(store, i, item, bar(kind + "F", i))
            i += 1
            if i == slots:
                i, ph = 0, ph ^ 1

    def turns_of(g):
        """(piece, block, tile, first, last, Q tile index, block index) of the group's turns."""
        x0, q0, n0, out = 0, 0, 0, []
        for n, (nb, tiles) in enumerate(plan):
            mine = (g - x0) & 1
            js = range(nb) if tiles == 2 else range(mine, nb, 2)
            for j in js:
                out.append((n, j, mine if tiles == 2 else 0, j == js[0], j == js[-1],
                            q0 + (mine if tiles == 2 else 0), n0 + j))
            x0, q0, n0 = x0 + nb * tiles, q0 + tiles, n0 + nb
        return out

    def issuer(g, kind):
        turns = turns_of(g)
        mma = mmas[2 * g + (kind == "PV")]
        seen = dict(Q=0, K=0, V=0)

        def see(name, slots, upto):
            """Waits for every copy up to this one in turn and releases those before it, which
            the other group alone uses: a parity cannot tell a phase from its next but one."""
            while seen[name] <= upto:
                i = seen[name] % slots
                if in_order or seen[name] == upto:
                    yield from wait(bar(name + "F", i), seen[name] // slots & 1)
                if seen[name] < upto:
                    bar(name + "E", i).arrive()
                seen[name] += 1

        ou = 0
        for x, (n, j, t, first, last, qn, kn) in enumerate(turns):
            buf = 2 * g + (x & 1)
            if kind == "S":
                qi, ki = qn % NQ, kn % NK
                if first:
                    yield from see("Q", NQ, qn)
                yield from see("K", NK, kn)
                yield from wait(bar("PV", buf), (x >> 1 & 1) ^ 1)

                def run(n=n, j=j, t=t, qi=qi, ki=ki, buf=buf):
                    assert q[qi] == (n, t) and k[ki] == (n, j)
                    assert s_buf[buf] in (None, "free")
                    s_buf[buf] = ("S", n, j, t)
                mma.append(run)
                mma.append(bar("S", buf).arrive)
                mma.append(bar("KE", ki).arrive)
                if last:
                    mma.append(bar("QE", qi).arrive)
            else:
                vi = kn % NV
                if first:
                    yield from wait(bar("OE", g), (ou & 1) ^ 1)
                yield from see("V", NV, kn)
                yield from wait(bar("P", buf), x >> 1 & 1)

                def run(n=n, j=j, t=t, vi=vi, first=first, buf=buf):
                    assert s_buf[buf] == ("P", n, j, t) and v[vi] == (n, j)
                    s_buf[buf] = "free"
                    if first:
                        assert o_buf[g] is None, "accumulator not read yet"
                        o_buf[g] = (n, [])
                    assert o_buf[g][0] == n
                    o_buf[g][1].append((j, t))
                    log.append((n, j, t))
                mma.append(run)
                mma.append(bar("PV", buf).arrive)
                mma.append(bar("VE", vi).arrive)
                ou += last

    read = {}

    def softmax(g, th):
        x0, turns, mu = 0, [0, 0], [0, 0]

        def turn_done(of, i):
            yield from wait(bar("PV", 2 * of + (i & 1)), i >> 1 & 1)

        for n, (nb, tiles) in enumerate(plan):
            mine = (g - x0) & 1
            for j in range(nb):
                if tiles == 1 and (j & 1) != mine:
                    continue
                x, buf = turns[g], 2 * g + (turns[g] & 1)
                turns[g] += 1
                yield from wait(bar("S", buf), x >> 1 & 1)
                want = (n, j, mine if tiles == 2 else 0)
                assert s_buf[buf] in (("S",) + want, ("P",) + want)
                yield
                if j > (tiles == 1) and rnd.random() < 0.3:  # the maximum moved: rescale O
                    yield from turn_done(g, x - 1)
                    assert o_buf[g][0] == n and o_buf[g][1][-1][0] == j - 3 + tiles
                s_buf[buf] = ("P",) + want
                bar("P", buf).arrive()
            if tiles == 2:
                turns[g ^ 1] += nb
                yield from turn_done(g, turns[g] - 1)
                assert o_buf[g] == (n, [(j, mine) for j in range(nb)])
                read.setdefault((n, g), set()).add((g, th))
                yield
                if len(read[(n, g)]) == 2:
                    o_buf[g] = None
                bar("OE", g).arrive(2)
            else:
                had = [nb > 1 or (x0 & 1) == i for i in range(2)]
                turns[g ^ 1] += (nb + mine) // 2
                if had[g]:
                    yield from turn_done(g, turns[g] - 1)
                    bar("ML", g).arrive()
                for i in range(2):
                    if had[i]:
                        yield from wait(bar("ML", i), mu[i] & 1)
                        yield from turn_done(i, turns[i] - 1)
                for i in range(2):
                    if had[i]:
                        assert o_buf[i] == (n, [(j, 0) for j in range(nb) if (x0 + j) & 1 == i])
                        read.setdefault((n, i), set()).add((g, th))
                yield
                for i in range(2):
                    if had[i]:
                        if len(read[(n, i)]) == 4:
                            o_buf[i] = None
                        bar("OE", i).arrive()
                        mu[i] += 1
            x0 += nb * tiles

    def tensor_core():
        while True:
            mma = rnd.choice(mmas)
            if mma:
                mma.pop(0)()
            yield

    kv = [(n, j) for n, (nb, _) in enumerate(plan) for j in range(nb)]
    def v_and_q():
        """V blocks; the next piece's Q with a piece's last block, before that block is waited
        for (a tail: every last block here)."""
        qs = [[(n, t) for t in range(tiles)] for n, (_, tiles) in enumerate(plan)]
        state = dict(q=0, v=0, t=0)

        def load_q():
            for item in qs.pop(0):
                i = state["q"] % NQ
                yield from wait(bar("QE", i), (state["q"] // NQ & 1) ^ 1)
                copy(q, i, item, bar("QF", i))
                state["q"] += 1

        yield from load_q()
        for n, (nb, _) in enumerate(plan):
            for j in range(nb):
                i = state["v"] % NV
                yield from wait(bar("VE", i), (state["v"] // NV & 1) ^ 1)
                tail = j + 2 >= nb  # waited for, made fit and released by this warp
                copy(v, i, (n, j), bar("VT", 0) if tail else bar("VF", i))
                if j + 1 == nb and qs:
                    yield from load_q()
                if tail:
                    yield from wait(bar("VT", 0), state["t"] & 1)
                    state["t"] += 1
                    bar("VF", i).arrive()
                state["v"] += 1

    roles = [issuer(g, kind) for g in range(2) for kind in ("S", "PV")]
    roles += [load("K", NK, k, kv), v_and_q()]
    roles += [softmax(g, th) for g in range(2) for th in range(2)]
    tc, cp = tensor_core(), copies()
    idle = 0
    while roles:
        i = rnd.randrange(len(roles) + 2)
        if i >= len(roles):
            next(tc if i == len(roles) else cp)
        else:
            try:
                next(roles[i])
            except StopIteration:
                roles.pop(i)
        idle += 1
        assert idle < 400 * (len(kv) + 10) * 40, "no end in sight"
    assert sorted(log) == [(n, j, t) for n, (nb, tiles) in enumerate(plan) for j in range(nb)
                           for t in range(tiles)]


@pytest.mark.parametrize("seed", range(120))
def test_turn_protocol(seed):
    r = random.Random(seed)
    plan = [(r.choice([1, 1, 2, 3, 4, 7]), r.choice([1, 2]) if seed % 3 == 0 else 1 + seed % 3 // 2)
            for _ in range(r.randint(1, 9))]
    protocol(plan, seed)


@pytest.mark.parametrize("seed", range(8))
def test_long_pieces_with_copies_out_of_order(seed):
    protocol([(40 + seed, 1), (3, 1), (25, 2), (1, 1), (30, 1)], seed)


def test_skipping_the_other_groups_copies_would_break_it():
    """An issuer that releases the other group's blocks unseen takes one phase for another."""
    broken = 0
    for seed in range(60):
        try:
            protocol([(40, 1), (31, 1)], seed, in_order=False)
        except AssertionError:
            broken += 1
    assert broken
