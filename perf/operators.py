"""Speculative decoding over the KV pool: what is measured of its three operators.

* attention for a tree of drafted tokens (``ops.attention_tree``, and with the
  nodes' K/V rows written first, ``ops.kv_append_attention_tree``);
* verification of the drafted tokens against the target's probabilities from
  given random numbers (``ops.verify_tree``);
* the move of the accepted path's rows to the end of the context
  (``ops.kv_commit``).

A tree has N nodes in an order in which a parent comes before its children:
``parents[b, i] < i``, -1 for a root.  Node i of sequence b sits in cache row
``seq_len[b] + i`` of the sequence's region; it sees the ``seq_len[b]`` context
rows, its ancestors and itself.
"""
import importlib
import random

import torch

own = False

HD = 128  # the head size of this framework's attention


def _ops():
    return importlib.import_module("nemotron-webgpu-decode_b200.ops")


# ------------------------------------------------------------------ cases

def _tree(name, batch, heads, kv_heads, nodes, lo, hi, append=False, ragged=False, chain=False,
          lens=1):
    """Attention: `batch` sequences of lo..hi context rows (drawn from `lens`)."""
    return {"name": name, "op": "tree", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "nodes": nodes, "lo": lo, "hi": hi, "append": append, "ragged": ragged,
            "chain": chain, "lens": lens}


def _verify(name, batch, nodes, vocab, draft=True, chain=False):
    return {"name": name, "op": "verify", "batch": batch, "nodes": nodes, "vocab": vocab,
            "draft": draft, "chain": chain}


def _commit(name, batch, nodes, pools, accepted, cap, kv_heads=8):
    return {"name": name, "op": "commit", "batch": batch, "nodes": nodes, "pools": pools,
            "accepted": accepted, "cap": cap, "kv_heads": kv_heads}


def listed():
    return [
        # the engine's own cache (256 rows) late in its 151-step trace: the latency of one user's step
        _tree("tree-engine", 1, 40, 8, 8, 150, 150, append=True),
        # one conversation of a few thousand tokens, a tree of two dozen drafts
        _tree("tree-one-4k", 1, 40, 8, 26, 4070, 4070),
        # one long document, the widest tree: 320 query rows per kv head share each K/V row
        _tree("tree-one-32k", 1, 40, 8, 64, 32768, 32768),
        # serving: the ragged lengths of the batched decode benchmark, a medium tree
        _tree("tree-batch-16", 64, 32, 8, 16, 512, 8192, lens=3),
        # serving with wide trees of differing sizes, K/V rows written in the same call
        _tree("tree-batch-61", 16, 40, 8, 61, 512, 8192, append=True, ragged=True, lens=5),
        # the batched decode benchmark's 256 sequences with a draft model's chain of four tokens
        _tree("chain-batch-5", 256, 32, 8, 5, 512, 8192, chain=True, lens=3),
        # one user, a chain of five drafts from a draft model, the model's own vocabulary
        _verify("verify-one", 1, 6, 131072, chain=True),
        # serving: trees sampled from a draft model
        _verify("verify-tree-32", 32, 26, 131072),
        # serving: many short chains
        _verify("verify-chain-256", 256, 5, 131072, chain=True),
        # drafts without probabilities (an n-gram table, the likeliest tokens), an odd vocabulary
        _verify("verify-points-64", 64, 16, 50257, draft=False),
        # one user: K and V of the engine's four attention layers, three tokens accepted
        _commit("commit-engine", 1, 8, 8, 3, 256),
        # serving: 128 sequences, four layers, wide trees
        _commit("commit-batch", 128, 64, 8, 9, 512),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.random()
    if kind < 0.6:
        while True:
            kv = rng.choice([1, 2, 4, 8])
            heads = kv * rng.choice([1, 2, 3, 4, 5, 5, 6, 7, 8])
            batch, nodes = _log_int(rng, 1, 256), _log_int(rng, 1, 64)
            hi = _log_int(rng, 1, 32768)
            lo = hi if rng.random() < 0.3 else rng.randint(0, hi)
            if batch * hi * kv <= 9_000_000 and batch * hi * nodes * heads <= 170_000_000 and \
                    batch * hi * nodes * heads >= 20_000:
                return dict(_tree("", batch, heads, kv, nodes, lo, hi, rng.random() < 0.4,
                                  rng.random() < 0.3, rng.random() < 0.3,
                                  rng.randint(1, 1 << 20)))
    if kind < 0.85:
        while True:
            batch, nodes, vocab = _log_int(rng, 1, 256), _log_int(rng, 1, 64), _log_int(rng, 1000, 160000)
            draft = rng.random() < 0.6
            if batch * nodes * vocab <= 160_000_000 and batch * nodes * nodes * vocab <= 3_000_000_000:
                return dict(_verify("", batch, nodes, vocab, draft, rng.random() < 0.4))
    batch, nodes = _log_int(rng, 1, 128), rng.randint(2, 64)
    accepted = rng.randint(1, max(1, min(nodes // 2, 9)))
    return dict(_commit("", batch, nodes, rng.choice([2, 4, 6, 8]), accepted,
                        rng.randint(128, 512), rng.choice([1, 2, 4, 8])))


def _lengths(case):
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def work(case):
    """Bytes and operations that one pass cannot do without."""
    if case["op"] == "tree":
        b, n, hq, kv = case["batch"], case["nodes"], case["heads"], case["kv_heads"]
        ctx = sum(_lengths(case))
        row = kv * HD * 2 * 2  # K and V of one cache row
        nbytes = (ctx + b * n) * row + 2 * b * n * hq * HD * 2
        if case["append"]:
            nbytes += b * n * row  # the new rows are read once and also written to the pool
        return {"bytes": nbytes, "flops": 4 * HD * hq * n * (ctx + b)}
    if case["op"] == "verify":
        # the row that the next token is drawn from (with its draft row where a draft was
        # rejected there, as at the end of most walks), and the drafted tokens' entries
        rows = 2 if case["draft"] else 1
        b = case["batch"]
        return {"bytes": b * (rows * case["vocab"] * 4 + case["nodes"] * (8 + 4 * rows)),
                "flops": b * case["vocab"] * rows}
    moved = case["batch"] * (case["accepted"] - 1) * case["pools"]
    return {"bytes": max(2 * moved * case["kv_heads"] * HD * 2, 4 * case["batch"] * case["nodes"]),
            "flops": 0}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _parents(case, r):
    """[batch, nodes]: a chain, or a bushy tree whose later nodes hang off recent ones."""
    out = []
    for _ in range(case["batch"]):
        row = [-1]
        for i in range(1, case["nodes"]):
            row.append(i - 1 if case["chain"] else r.randint(max(0, (i - 1) // 3 - 2), (i - 1) // 2))
        out.append(row)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"tree": _prepare_tree, "verify": _prepare_verify, "commit": _prepare_commit}[case["op"]](
        case, seed)


def _prepare_tree(case, seed):
    g, r = _gen(seed), random.Random(seed)
    b, n, hq, kv = case["batch"], case["nodes"], case["heads"], case["kv_heads"]
    lens = _lengths(case)
    offs, rows = [], 0
    for length in lens:  # each sequence's region holds its context, its tree and a few spare rows
        offs.append(rows)
        rows += length + n + 3

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)

    s = {"op": "tree", "hq": hq, "kv": kv, "k": normal(rows, kv, HD), "v": normal(rows, kv, HD),
         "q": normal(b, n, hq, HD),
         "row_offset": torch.tensor(offs, dtype=torch.int64, device="cuda"),
         "seq_len": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "max_rows": max(lens) + n, "parents": _parents(case, r), "tree_len": None,
         "k_new": None, "v_new": None, "o": torch.empty(b, n, hq, HD, dtype=torch.float16, device="cuda")}
    if case["ragged"]:
        s["tree_len"] = torch.tensor([r.randint(1, n) for _ in range(b)], dtype=torch.int32,
                                     device="cuda")
    if case["append"]:
        s["k_new"], s["v_new"] = normal(b, n, kv, HD), normal(b, n, kv, HD)
    return s


def _prepare_verify(case, seed):
    g, r = _gen(seed), random.Random(seed)
    b, n, vocab = case["batch"], case["nodes"], case["vocab"]
    parents = _parents(case, r)
    # a target that has made up its mind to a degree, a draft model that is near it
    logits = torch.randn(b, n, vocab, generator=g, device="cuda") * 3.0
    target = torch.softmax(logits, -1)
    logits += torch.randn(b, n, vocab, generator=g, device="cuda")
    draft = torch.softmax(logits, -1)
    del logits
    at = parents.clamp(min=0).long()  # node i's token was drawn from its parent's draft row
    rows = at + torch.arange(b, device="cuda")[:, None] * n
    if case["draft"]:
        tokens = torch.multinomial(draft.view(b * n, vocab).index_select(0, rows.view(-1)), 1,
                                   generator=g)
    else:  # the likeliest tokens of the draft, the k-th of them for the k-th node
        top = draft.topk(min(n, vocab), -1).indices.view(b * n, -1)
        tokens = top[rows.view(-1), torch.arange(n, device="cuda").repeat(b) // 2]
        draft = None
    return {"op": "verify", "tokens": tokens.view(b, n).int(), "parents": parents,
            "target": target, "draft": draft,
            "u": torch.rand(b, n, generator=g, device="cuda"),
            "w": torch.rand(b, generator=g, device="cuda")}


def _prepare_commit(case, seed):
    g, r = _gen(seed), random.Random(seed)
    b, n, cap, kv, acc = (case[k] for k in ("batch", "nodes", "cap", "kv_heads", "accepted"))
    path = torch.full((b, n), -1, dtype=torch.int32)
    for i in range(b):
        # the accepted nodes come after the rows that they move to (the path's first node stays)
        path[i, :acc] = torch.tensor([0] + sorted(r.sample(range(acc, n), acc - 1)),
                                     dtype=torch.int32)
    return {"op": "commit",
            "pools": [torch.randn(b * cap, kv, HD, generator=g, device="cuda", dtype=torch.float16)
                      for _ in range(case["pools"])],
            "row_offset": torch.arange(b, device="cuda", dtype=torch.int64) * cap,
            "pos": torch.tensor([r.randint(0, cap - n) for _ in range(b)], dtype=torch.int32,
                                device="cuda"),
            "path": path.cuda(),
            "n_accepted": torch.full((b,), acc, dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    return {"tree": _plain_tree, "verify": _plain_verify, "commit": _plain_commit}[s["op"]](s)


def _run_own(s):
    ops = _ops()
    if s["op"] == "tree":
        if s["k_new"] is None:
            ops.attention_tree(s["q"], s["k"], s["v"], s["row_offset"], s["seq_len"], s["parents"],
                               s["o"], s["hq"], s["kv"], HD, tree_len=s["tree_len"])
            return {"o": s["o"]}
        ops.kv_append_attention_tree(s["q"], s["k_new"], s["v_new"], s["k"], s["v"],
                                     s["row_offset"], s["seq_len"], s["parents"], s["o"], s["hq"],
                                     s["kv"], HD, tree_len=s["tree_len"])
        return {"o": s["o"], "k": s["k"], "v": s["v"]}
    if s["op"] == "verify":
        path, n_accepted, token = ops.verify_tree(s["tokens"], s["parents"], s["target"], s["u"],
                                                  s["w"], draft_probs=s["draft"])
        return {"path": path, "n_accepted": n_accepted, "token": token}
    ops.kv_commit(s["pools"], s["row_offset"], s["pos"], s["path"], s["n_accepted"])
    return {"pools": s["pools"]}


def _present(s, b, n):
    node = torch.arange(n, device="cuda")
    if s["tree_len"] is None:
        return torch.ones(b, n, dtype=torch.bool, device="cuda")
    return node[None] < s["tree_len"][:, None]


def _plain_tree(s):
    b, n, hq, _ = s["q"].shape
    kv, g, span = s["kv"], s["hq"] // s["kv"], s["max_rows"]
    node = torch.arange(n, device="cuda")
    present = _present(s, b, n)
    if s["k_new"] is not None:
        rows = (s["row_offset"] + s["seq_len"])[:, None] + node
        s["k"][rows[present]] = s["k_new"][present]
        s["v"][rows[present]] = s["v_new"][present]
    # which nodes a node descends from: the powers of (identity + parent links)
    link = (s["parents"].long()[:, :, None] == node).float()
    sees = torch.matrix_power(link + torch.eye(n, device="cuda"), n) > 0
    # every sequence's rows side by side, in 32 bits
    t = torch.arange(span, device="cuda")
    rows = (s["row_offset"][:, None] + t).clamp(max=s["k"].shape[0] - 1)
    k = s["k"][rows].float().permute(0, 2, 3, 1)
    v = s["v"][rows].float().permute(0, 2, 1, 3)
    q = s["q"].float().view(b, n, kv, g, HD).permute(0, 2, 1, 3, 4).reshape(b, kv, n * g, HD)
    scores = torch.matmul(q * HD ** -0.5, k).view(b, kv, n, g, span)
    after = t - s["seq_len"][:, None].long()  # row t's place in the tree
    seen = torch.gather(sees, 2, after.clamp(0, n - 1)[:, None].expand(b, n, span))
    seen = (after < 0)[:, None] | (seen & (after < n)[:, None])
    scores = scores.masked_fill(~seen[:, None, :, None], float("-inf"))
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    scores = scores / scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(b, kv, n * g, span), v)
    o = o.view(b, kv, n, g, HD).permute(0, 2, 1, 3, 4).reshape(b, n, hq, HD)
    o = torch.where(present[:, :, None, None], o, torch.zeros((), device="cuda")).half()
    if s["k_new"] is not None:
        return {"o": o, "k": s["k"], "v": s["v"]}
    return {"o": o}


def _plain_verify(s):
    b, n, vocab = s["target"].shape
    every = torch.arange(b, device="cuda")
    parents, tokens = s["parents"].long(), s["tokens"].long()
    cur = torch.zeros(b, dtype=torch.long, device="cuda")  # the last accepted node
    count = torch.ones_like(cur)
    path = torch.full((b, n), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    rest = s["target"][:, 0].double()  # what is left of the row at `cur`
    for c in range(1, n):
        child = parents[:, c] == cur
        tok = tokens[:, c]
        u = s["u"][:, c].double()
        if s["draft"] is not None:
            q = s["draft"][every, cur].double()
            passed = child & (u * q[every, tok] < rest[every, tok])
            less = (rest - q).clamp(min=0)
        else:
            passed = child & (u < rest[every, tok])
            less = rest.clone()
            less[every, tok] = 0
        total = less.sum(-1, keepdim=True)
        whole = s["target"][every, cur].double()
        less = torch.where(total > 0, less / total, whole)  # nothing left: the whole row again
        rest = torch.where((child & ~passed)[:, None], less, rest)
        rest = torch.where(passed[:, None], s["target"][:, c].double(), rest)
        cur = torch.where(passed, c, cur)
        at = count.clamp(max=n - 1)
        path[every, at] = torch.where(passed, c, path[every, at].long()).int()
        count = count + passed
    cum = rest.cumsum(-1)
    hit = cum > (s["w"].double()[:, None] * cum[:, -1:])
    return {"path": path, "n_accepted": count.int(), "token": hit.int().argmax(-1).int()}


def _plain_commit(s):
    b, n = s["path"].shape
    j = torch.arange(n, device="cuda")
    moves = j[None] < s["n_accepted"][:, None]
    base = (s["row_offset"] + s["pos"])[:, None]
    src, dst = (base + s["path"])[moves], (base + j)[moves]
    for pool in s["pools"]:
        pool[dst] = pool[src]
    return {"pools": s["pools"]}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """Outputs from the definitions, a sequence at a time, in 64 bits; moved rows have none."""
    s = prepare(case, seed)
    if case["op"] == "commit":
        return None
    if case["op"] == "verify":
        return _exact_verify(s)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    b, n, hq, _ = s["q"].shape
    g = hq // s["kv"]
    lens, offs, parents = s["seq_len"].tolist(), s["row_offset"].tolist(), s["parents"].tolist()
    sizes = [n] * b if s["tree_len"] is None else s["tree_len"].tolist()
    for i in range(b):
        m, ctx, off = sizes[i], lens[i], offs[i]
        k, v = s["k"][off:off + ctx + m].double(), s["v"][off:off + ctx + m].double()
        if s["k_new"] is not None:
            k[ctx:], v[ctx:] = s["k_new"][i, :m].double(), s["v_new"][i, :m].double()
        bias = torch.zeros(m, ctx + m, dtype=torch.float64)
        bias[:, ctx:] = -float("inf")
        for node in range(m):
            up = node
            while up >= 0:
                bias[node, ctx + up] = 0
                up = parents[i][up]
        for h in range(hq):
            score = s["q"][i, :m, h].double() @ k[:, h // g].T / HD ** 0.5 + bias.cuda()
            out[i, :m, h] = torch.softmax(score, -1) @ v[:, h // g]
    return {"o": out} if s["k_new"] is None else {"o": out, "k": None, "v": None}


def _exact_verify(s):
    b, n, _ = s["target"].shape
    parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
    us, ws = s["u"].tolist(), s["w"].tolist()
    paths, counts, drawn = [], [], []
    for i in range(b):
        walk, going = [0], True
        while going:
            at, going = walk[-1], False
            p = s["target"][i, at].double()
            for c in [c for c in range(1, n) if parents[i][c] == at]:
                t = tokens[i][c]
                q = torch.zeros_like(p) if s["draft"] is None else s["draft"][i, at].double()
                if s["draft"] is None:
                    q[t] = 1.0
                if us[i][c] * q[t].item() < p[t].item():
                    walk.append(c)
                    going = True
                    break
                left = torch.maximum(p - q, torch.zeros_like(p))
                if s["draft"] is None:
                    left[t] = 0.0
                mass = left.sum()
                p = left / mass if mass > 0 else s["target"][i, at].double()
        below = torch.cumsum(p, 0)
        drawn.append(int(torch.nonzero(below > ws[i] * below[-1])[0, 0]))
        counts.append(len(walk))
        paths.append(walk + [-1] * (n - len(walk)))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"path": as_int(paths), "n_accepted": as_int(counts), "token": as_int(drawn)}
