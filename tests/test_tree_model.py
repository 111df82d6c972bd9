"""CPU models of the tree-attention kernel's work split and of its turn protocol
(csrc/tree_attn.cu), which cannot be looked into on the GPU.

* the split: the CTAs' pieces cover every unit's blocks once, every unit that a cut divides
  has exactly one joining CTA, whose piece list is the unit's, and no partial slot is used twice;
* the protocol: MMA issuer, producers and the two softmax groups, with mbarriers that only
  know the parity of their phase, run under random timing to the end, each turn's softmax
  reads the scores of its own block, and no accumulator or stage is overwritten in use.
"""
from __future__ import annotations

import random

import pytest

BN = 128


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


def protocol(plan, seed, NQ=2, NK=3, NV=2):
    """plan: [(nb, tiles)] per piece.  Roles are generators that yield until a wait passes."""
    rnd = random.Random(seed)
    bars = {}

    def bar(name, i, count=1):
        return bars.setdefault((name, i), Bar(count))

    for g in range(2):
        bar("P", g, 2), bar("OE", g, 4), bar("ML", g, 2)  # two threads stand for a group's 128
    q, k, v = [None] * NQ, [None] * NK, [None] * NV
    s_buf, o_buf, log = [None, None], [None, None], []
    mma = []  # issued, not yet run: (function) in order

    def wait(b, parity):
        while not b.passed(parity):
            yield

    def load(kind, slots, store, items):
        i, ph = 0, 0
        for item in items:
            yield from wait(bar(kind + "E", i), ph ^ 1)
            store[i] = item
            yield
            bar(kind + "F", i).arrive()
            i += 1
            if i == slots:
                i, ph = 0, ph ^ 1

    def issuer():
        turns = [(n, j, t, tiles, nb) for n, (nb, tiles) in enumerate(plan) for j in range(nb)
                 for t in range(tiles)]
        st = dict(q=0, qp=0, qpiece=(0, 0), k=0, kp=0, x=0)

        def issue_s():
            n, j, t, tiles, nb = turns[st["x"]]
            g = st["x"] & 1
            if t == 0:
                if j == 0:
                    st["qpiece"] = (st["q"], st["qp"])
                st["q"], st["qp"] = st["qpiece"]
            if j == 0:
                yield from wait(bar("QF", st["q"]), st["qp"])
            yield from wait(bar("KF", st["k"]), st["kp"])
            qi, ki = st["q"], st["k"]

            def run():
                assert q[qi] == (n, t) and k[ki] == (n, j)
                s_buf[g] = ("S", n, j, t)
            mma.append(run)
            mma.append(lambda: bar("S", g).arrive())
            if j + 1 == nb:
                mma.append(lambda: bar("QE", qi).arrive())
            st["q"] += 1
            if st["q"] == NQ:
                st["q"], st["qp"] = 0, st["qp"] ^ 1
            st["x"] += 1
            if t + 1 == tiles:
                mma.append(lambda: bar("KE", ki).arrive())
                st["k"] += 1
                if st["k"] == NK:
                    st["k"], st["kp"] = 0, st["kp"] ^ 1

        for _ in range(min(2, len(turns))):
            yield from issue_s()
        vi, vp, pp, ou = 0, 0, [0, 0], [0, 0]
        for x, (n, j, t, tiles, nb) in enumerate(turns):
            g = x & 1
            first = j == 0 if tiles == 2 else j < 2
            last = j + 1 == nb if tiles == 2 else j + 2 >= nb
            if first:
                yield from wait(bar("OE", g), (ou[g] & 1) ^ 1)
            yield from wait(bar("P", g), pp[g])
            yield from wait(bar("VF", vi), vp)

            def run(g=g, n=n, j=j, t=t, vi=vi, first=first):
                assert s_buf[g] == ("P", n, j, t) and v[vi] == (n, j)
                if first:
                    assert o_buf[g] is None, "accumulator not read yet"
                    o_buf[g] = (n, [])
                assert o_buf[g][0] == n
                o_buf[g][1].append((j, t))
                log.append((n, j, t))
            mma.append(run)
            if last:
                mma.append(lambda g=g: bar("OF", g).arrive())
                ou[g] += 1
            pp[g] ^= 1
            if t + 1 == tiles:
                mma.append(lambda vi=vi: bar("VE", vi).arrive())
                vi += 1
                if vi == NV:
                    vi, vp = 0, vp ^ 1
            if st["x"] < len(turns):
                yield from issue_s()

    read = {}

    def softmax(g, th):
        sp, x0, ou, mu = 0, 0, [0, 0], [0, 0]
        for n, (nb, tiles) in enumerate(plan):
            mine = (g - x0) & 1
            for j in range(nb):
                if tiles == 1 and (j & 1) != mine:
                    continue
                yield from wait(bar("S", g), sp)
                sp ^= 1
                want = (n, j, mine if tiles == 2 else 0)
                assert s_buf[g] in (("S",) + want, ("P",) + want)
                yield
                s_buf[g] = ("P",) + want
                bar("P", g).arrive()
            if tiles == 2:
                yield from wait(bar("OF", g), ou[g] & 1)
                assert o_buf[g] == (n, [(j, mine) for j in range(nb)])
                read.setdefault((n, g), set()).add((g, th))
                yield
                if len(read[(n, g)]) == 2:
                    o_buf[g] = None
                bar("OE", g).arrive(2)
                ou[0] += 1
                ou[1] += 1
            else:
                had = [nb > 1 or (x0 & 1) == i for i in range(2)]
                if had[g]:
                    bar("ML", g).arrive()
                for i in range(2):
                    if had[i]:
                        yield from wait(bar("ML", i), mu[i] & 1)
                        yield from wait(bar("OF", i), ou[i] & 1)
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
                        ou[i] += 1
                        mu[i] += 1
            x0 += nb * tiles

    def tensor_core():
        while True:
            if mma:
                mma.pop(0)()
            yield

    kv = [(n, j) for n, (nb, _) in enumerate(plan) for j in range(nb)]
    roles = [issuer(), load("K", NK, k, kv), load("V", NV, v, kv),
             load("Q", NQ, q, [(n, t) for n, (_, tiles) in enumerate(plan) for t in range(tiles)])]
    roles += [softmax(g, th) for g in range(2) for th in range(2)]
    tc = tensor_core()
    idle = 0
    while roles:
        i = rnd.randrange(len(roles) + 1)
        if i == len(roles):
            next(tc)
        else:
            try:
                next(roles[i])
            except StopIteration:
                roles.pop(i)
        idle += 1
        assert idle < 400 * (len(kv) + 10) * 40, "no end in sight"
    assert log == [(n, j, t) for n, (nb, tiles) in enumerate(plan) for j in range(nb)
                   for t in range(tiles)]


@pytest.mark.parametrize("seed", range(40))
def test_turn_protocol(seed):
    r = random.Random(seed)
    plan = [(r.choice([1, 1, 2, 3, 4, 7]), r.choice([1, 2]) if seed % 3 == 0 else 1 + seed % 3 // 2)
            for _ in range(r.randint(1, 9))]
    protocol(plan, seed)
