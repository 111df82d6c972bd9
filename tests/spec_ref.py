"""Plain 64-bit restatements of the speculative-decoding operators, a sequence at a time."""
from __future__ import annotations

import numpy as np


def random_parents(rng, n, chain=False, roots=False):
    """parents[i] < i; node 0 is a root, others too where `roots`."""
    if chain:
        return np.arange(-1, n - 1, dtype=np.int32)
    low = -1 if roots else 0
    return np.array([-1] + [rng.integers(max(low, i - 6), i) for i in range(1, n)], dtype=np.int32)


def ancestors(parents, i):
    seen = []
    while i >= 0:
        seen.append(i)
        i = int(parents[i])
    return seen


def tree_attention(q, k, v, ctx, parents, m, n_kv, scale):
    """q [N, Hq, hd], k / v [ctx + m, n_kv, hd] f64 -> (o [N, Hq, hd], a bound's parts):
    mag = sum of p |v| per element, amp = max over the attended rows of sum |q_d k_d|."""
    n, hq, hd = q.shape
    g = hq // n_kv
    o, mag, amp = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for i in range(m):
        rows = list(range(ctx)) + sorted(ctx + a for a in ancestors(parents, i))
        kk, vv = k[rows], v[rows]
        for h in range(n_kv):
            s = q[i, h * g:(h + 1) * g] @ kk[:, h].T * scale
            with np.errstate(invalid="ignore"):
                amp = max(amp, float(np.max(np.abs(q[i, h * g:(h + 1) * g]) @ np.abs(kk[:, h]).T)))
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o[i, h * g:(h + 1) * g] = p @ vv[:, h]
            mag[i, h * g:(h + 1) * g] = p @ np.abs(vv[:, h])
    return o, mag, amp


def attention_bound(o, mag, amp, rows, scale, vmax):
    """How far an fp16 output may be from the 64-bit one, element by element.

    Output rounding: half a step, 2^-11 |o|, or 2^-25 below the normal range.
    Weights: a score is a sum of 128 products in f32, off by at most 128 * 2^-24 of
    sum |q k|, so exp is off by twice that much of itself (numerator and denominator);
    a weight is rounded to fp16 once, 2^-11 of itself, or below the normal range
    2^-25 against a largest weight of at least 2^7 (each row, against the sum);
    exp2 and the scaling 2^-21.  Sums of `rows` terms in f32: rows * 2^-24 twice.
    """
    ds = 128 * 2.0 ** -24 * amp * scale
    w = 2.0 ** -11 + 2 * ds + 2.0 ** -20 + 2 * (rows + 8) * 2.0 ** -24
    return 2.0 ** -11 * np.abs(o) * (1 + w) + w * mag + rows * 2.0 ** -32 * vmax + 2.0 ** -25


def verify(tokens, parents, m, target, draft, u, w):
    """One sequence: (path, next token).  Probabilities f32 arrays [N, V]."""
    if m == 0:
        return [], -1
    at, path = 0, [0]

    def row(x):
        x = x.astype(np.float64)
        return np.where(x > 0, x, 0.0)

    vocab = target.shape[1]
    while True:
        r, accepted = row(target[at]), None
        for c in range(1, m):
            if parents[c] != at:
                continue
            t = int(tokens[c])
            inside = 0 <= t < vocab
            if draft is not None:
                q = row(draft[at])
                if inside and float(u[c]) * q[t] < r[t]:
                    accepted = c
                    break
                r = np.maximum(r - q, 0.0)
            else:
                if inside and float(u[c]) < r[t]:
                    accepted = c
                    break
                r = r.copy()
                if inside:
                    r[t] = 0.0
            total = r.sum()
            r = r / total if total > 0 else row(target[at])
        if accepted is None:
            cum = np.cumsum(r)
            if not cum[-1] > 0:
                return path, -1
            return path, int(np.argmax(cum > float(w) * cum[-1]))
        path.append(accepted)
        at = accepted
