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


def unit_tiles(u, n_tiles):
    per_head = -(-n_tiles // 2)
    return 2 if (u % per_head) * 2 + 1 < n_tiles else 1


UNIT_BLOCKS, MIN_BLOCKS = 6, 4


def one_sequence(nblk, n_kv, n_tiles, ctas, cost1, cost2):
    """The split of a single sequence, or None where the batch's is used."""
    per_head, pairs, single = -(-n_tiles // 2), n_tiles // 2, n_tiles % 2
    head_ctas = ctas // n_kv
    if head_ctas < per_head:
        return None
    k1 = max(1, head_ctas * cost1 // (pairs * cost2 + single * cost1)) if single else 0
    k2 = (head_ctas - k1) // pairs if pairs else 0
    k1 = head_ctas - pairs * k2 if single else 0
    out, joins = [], {}
    for c in range(ctas):
        head, i = divmod(c, head_ctas)
        k, unit, at = k2, i // k2 if pairs else 0, i % k2 if pairs else i
        if unit >= pairs:
            unit, at, k = pairs, i - pairs * k2, k1
        mine = []
        out.append(mine)
        if head < n_kv and unit < per_head and at < k:
            k = max(1, min(k, nblk // MIN_BLOCKS))
            if at < k:
                lo, hi = nblk * at // k, nblk * (at + 1) // k
                mine.append((0, head * per_head + unit, lo, hi - lo))
                if at > 0 and at + 1 == k:
                    joins[c] = (0, head * per_head + unit, c - at)
    return out, joins, n_kv * per_head


def pieces(blocks, n_kv, tiles, ctas, cost1, cost2):
    """Per CTA the list of (b, u, blk, nb) and its join (b, u, first), as the kernel finds them;
    `tiles`: those of each sequence's present nodes."""
    if len(blocks) == 1:
        split = one_sequence(blocks[0], n_kv, tiles[0], ctas, cost1, cost2)
        if split:
            return split
    head_cost = [t // 2 * cost2 + t % 2 * cost1 for t in tiles]
    length = [(n + UNIT_BLOCKS) * h for n, h in zip(blocks, head_cost)]
    total = sum(length) * n_kv
    per = max(-(-total // ctas), cost2)
    cost_of = lambda b, u: cost2 if unit_tiles(u, tiles[b]) == 2 else cost1  # noqa: E731
    out, joins = [], {}
    for c in range(ctas):
        x0, x1 = min(total, c * per), min(total, c * per + per)
        mine = []
        out.append(mine)
        if x0 >= x1:
            continue
        y, lo, b = x0 // n_kv, 0, 0
        while not lo <= y < lo + length[b]:
            lo += length[b]
            b += 1
        n, per_head = blocks[b], -(-tiles[b] // 2)
        r = x0 - lo * n_kv
        head, r = divmod(r, length[b])
        k = min(r // ((n + UNIT_BLOCKS) * cost2), per_head - 1)
        r -= k * (n + UNIT_BLOCKS) * cost2
        start, u = x0 - r, head * per_head + k
        cost = cost_of(b, u)
        blk = -(-r // cost)
        if blk < n:
            left = x1 - start - blk * cost
            if blk > 0 and left > 0 and blk + -(-left // cost) >= n:
                joins[c] = (b, u, start // per)
        else:
            left = x1 - start - (n + UNIT_BLOCKS) * cost
            blk = n
        while left > 0:
            if blk == n:
                blk, u = 0, u + 1
                if u == n_kv * -(-tiles[b] // 2):
                    u, b = 0, b + 1
                n = blocks[b]
            cost = cost_of(b, u)
            nb = n - blk if left >= (n - blk) * cost else -(-left // cost)
            mine.append((b, u, blk, nb))
            blk += nb
            left -= (nb + (UNIT_BLOCKS if blk == n else 0)) * cost
    return out, joins, n_kv * sum(-(-t // 2) for t in tiles)


@pytest.mark.parametrize("seed", range(120))
def test_split_covers_every_unit(seed):
    r = random.Random(seed)
    blocks = [r.choice([1, 1, 2, 5, 33, r.randint(1, 400)]) for _ in range(r.choice([1, 1, 2, 7, 64]))]
    cost1 = r.choice([1, 1, 2, 3])
    n_tiles = r.choice([1, 2, 3, 4])
    tiles = [r.choice([n_tiles, r.randint(1, n_tiles)]) for _ in blocks]
    got, joins, n_units = pieces(blocks, r.choice([1, 2, 8]), tiles, r.choice([1, 7, 148]), cost1,
                                 r.randint(cost1, 2 * cost1))
    seen, slots = {}, set()
    for c, mine in enumerate(got):
        for b, u, blk, nb in mine:
            assert nb > 0
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
    assert len(seen) == n_units


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
        bar("P", 2 * g, 2), bar("P", 2 * g + 1, 2), bar("OE", g, 2), bar("ML", g, 2)  # two threads stand for a group's 128
    q, k, v = [None] * NQ, [None] * NK, [None] * NV
    s_buf, o_buf, log = [None] * 4, [None, None], []
    mmas = [[], [], [], []]  # issued by an issuer, not yet run, in order

    def wait(b, parity):
        while not b.passed(parity):
            yield

    NP, USERS = 4, 13
    for i in range(NP):
        bar("PCE", i, USERS)

    def planner():
        for n in range(len(plan) + 1):  # the last one says that there are no more
            yield from wait(bar("PCE", n % NP), (n // NP & 1) ^ 1)
            bar("PCF", n % NP).arrive()

    def get(n):
        yield from wait(bar("PCF", n % NP), n // NP & 1)
        bar("PCE", n % NP).arrive()

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
        i, ph, piece = 0, 0, -1
        for item in items:
            if item[0] != piece:
                piece = item[0]
                yield from get(piece)
            yield from wait(bar(kind + "E", i), ph ^ 1)
            copy(store, i, item, bar(kind + "F", i))
            i += 1
            if i == slots:
                i, ph = 0, ph ^ 1
        yield from get(len(plan))

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

        ou, got = 0, 0
        for x, (n, j, t, first, last, qn, kn) in enumerate(turns):
            buf = 2 * g + (x & 1)
            while got <= n:
                yield from get(got)
                got += 1
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
        while got <= len(plan):
            yield from get(got)
            got += 1

    read, handed = {}, [[None, None], [None, None]]  # [group][thread]

    def softmax(g, th):
        x0, turn, units = 0, 0, 0
        for n, (nb, tiles) in enumerate(plan):
            yield from get(n)
            mine, first = (g - x0) & 1, turn
            for j in range(nb) if tiles == 2 else range(mine, nb, 2):
                x, buf = turn, 2 * g + (turn & 1)
                turn += 1
                yield from wait(bar("S", buf), x >> 1 & 1)
                want = (n, j, mine if tiles == 2 else 0)
                assert s_buf[buf] in (("S",) + want, ("P",) + want)
                yield
                if x != first and rnd.random() < 0.3:  # the maximum moved: rescale O
                    yield from wait(bar("PV", 2 * g + (x - 1 & 1)), x - 1 >> 1 & 1)
                    assert o_buf[g][0] == n and o_buf[g][1][-1][0] == j - 3 + tiles
                s_buf[buf] = ("P",) + want
                bar("P", buf).arrive()
            x0 += nb * tiles
            if turn != first:
                yield from wait(bar("OE", g), (units & 1) ^ 1)
                units += 1
                assert handed[g][th] is None
                handed[g][th] = n
                bar("ML", g).arrive()
        yield from get(len(plan))

    def epilogue(th):
        x0, turns, units = 0, [0, 0], [0, 0]

        def complete(i):
            yield from wait(bar("ML", i), units[i] & 1)
            last = turns[i] - 1
            yield from wait(bar("PV", 2 * i + (last & 1)), last >> 1 & 1)

        for n, (nb, tiles) in enumerate(plan):
            yield from get(n)
            lead = x0 & 1
            own = {0: nb, 1: nb} if tiles == 2 else {lead: (nb + 1) // 2, lead ^ 1: nb // 2}
            groups = [i for i in (own if tiles == 2 else (lead, lead ^ 1)) if own[i]]
            for i in groups:
                turns[i] += own[i]
            for part in [[i] for i in groups] if tiles == 2 else [groups]:
                for i in part:
                    yield from complete(i)
                for i in part:
                    js = [(j, (i - x0) & 1) for j in range(nb)] if tiles == 2 else \
                        [(j, 0) for j in range(nb) if (x0 + j) & 1 == i]
                    assert o_buf[i] == (n, js) and handed[i][th] == n
                yield
                for i in part:
                    handed[i][th] = None
                    read.setdefault((n, i), set()).add(th)
                    if len(read[(n, i)]) == 2:
                        o_buf[i] = None
                    bar("OE", i).arrive()
                    units[i] += 1
            x0 += nb * tiles
        yield from get(len(plan))

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
        state = dict(q=0, v=0)

        def load_q(block=True):
            while qs[0]:
                i, parity = state["q"] % NQ, (state["q"] // NQ & 1) ^ 1
                if not block and not bar("QE", i).passed(parity):
                    return
                yield from wait(bar("QE", i), parity)
                copy(q, i, qs[0].pop(0), bar("QF", i))
                state["q"] += 1

        yield from get(0)
        yield from load_q()
        qs.pop(0)
        for n, (nb, _) in enumerate(plan):
            yield from get(n + 1)
            for j in range(nb):
                i = state["v"] % NV
                yield from wait(bar("VE", i), (state["v"] // NV & 1) ^ 1)
                tail = j + 2 >= nb  # made fit and released by another warp
                copy(v, i, (n, j), bar("VT", i) if tail else bar("VF", i))
                state["v"] += 1
                if qs:
                    yield from load_q(j + 1 == nb)
            if qs:
                qs.pop(0)

    def tails():
        phases, i = [0] * NV, 0
        for n, (nb, _) in enumerate(plan):
            yield from get(n)
            for j in range(nb):
                if j + 2 >= nb:
                    yield from wait(bar("VT", i), phases[i])
                    phases[i] ^= 1
                    yield
                    bar("VF", i).arrive()
                i = (i + 1) % NV
        yield from get(len(plan))

    roles = [issuer(g, kind) for g in range(2) for kind in ("S", "PV")]
    roles += [load("K", NK, k, kv), v_and_q(), tails(), planner()] + [epilogue(th) for th in range(2)]
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
