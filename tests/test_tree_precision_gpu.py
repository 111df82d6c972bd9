"""Tree attention within the parity tolerance that the decode path keeps (tolerance.py):
max-abs 2e-3 and, where outputs average out to nearly nothing, max-rel 1e-2.

What the kernels may add to the 64-bit value for N(0, 1) inputs: the output's rounding, 2^-11 of
it; a weight as fp16 head and remainder, 2^-22 of it or 2^-32 of the largest; a score's sum of
128 products in f32, at random some 2^-22 of sum |q k| scale (about 7), so 2e-6 of a weight.
With sum p |v| about 0.8 that is 2e-6 against an element of 1e-3: 0.2 % and the rounding's
0.05 %, a quarter of the tolerance.  One fp16 rounding of the weights alone, 2^-11 each at
random over some hundred rows that count, is 1e-5 to 2e-5 and breaks it.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from devutil import vals
from spec_ref import tree_attention
from test_tree_gpu import HD, Case, _attend
from tolerance import assert_attn_close

pytestmark = pytest.mark.gpu


def _reference(c, b, nodes):
    lo, hi = c.off[b], c.off[b] + c.ctx[b] + c.m[b]
    q = np.zeros((c.n, c.nh, HD))
    q[nodes] = c.q[b, nodes]
    ref, _, _ = tree_attention(q, c.k[lo:hi].astype(np.float64), c.v[lo:hi].astype(np.float64),
                               c.ctx[b], c.parents[b], c.m[b], c.nkv, HD ** -0.5)
    return ref[nodes]


@pytest.mark.parametrize("ctx,n,nh,nkv", [
    ([4096], 64, 40, 8),            # three tiles, split over the processors
    ([4096], 5, 40, 8),             # few query rows
    ([1500, 4000, 700], 26, 16, 2), # a batch: units of two tiles and their ends
    ([900] * 30, 4, 32, 8),
    ([1900], 12, 40, 8),            # a small pool: a cluster per head
    ([90], 8, 40, 8),               # ... one CTA
])
@pytest.mark.parametrize("chain", [False, True])
def test_parity_tolerance(ops, ctx, n, nh, nkv, chain):
    c = Case(ctx, n, nh, nkv, seed=sum(ctx) + n, chain=chain)
    got = vals(_attend(ops, c.dev(), nh, nkv))
    for b in range(min(c.b, 3)):
        assert_attn_close(got[b], _reference(c, b, list(range(n))), f"sequence {b}")


@pytest.mark.parametrize("ctx,n", [(4096, 7), (1700, 7), (100, 7)])
def test_chain_gives_what_decode_steps_give(ops, ctx, n):
    """Each of the two within the tolerance of the formula, and of the other."""
    c = Case([ctx], n, 40, 8, seed=ctx, chain=True, guard=0)
    d = c.dev()
    got, ref = vals(_attend(ops, d, 40, 8))[0], _reference(c, 0, list(range(n)))
    for i in range(n):
        o = torch.empty(40, HD, dtype=torch.float16, device="cuda")
        ops.attention(d["q"][0, i].contiguous(), d["k_pool"], d["v_pool"], o,
                      ops.AttnParams(40, 8, HD, ctx + i + 1))
        assert_attn_close(got[i], ref[i], f"node {i}")
        assert_attn_close(got[i], vals(o), f"node {i} against the step")


@pytest.mark.parametrize("ctx", [2000, 16000])
@pytest.mark.parametrize("log2", [15, 20, 22])
def test_small_weights_in_great_number(ops, ctx, log2):
    """A tail of equal weights of 2^-log2 of the largest, which alone has an output (V of the
    large row is zero).  A weight is off by 2^-32 of the largest at most (the general kernel's
    largest is at least 2^7, an fp16 step below the normal range 2^-24, half of it the rounding),
    the sum by that much of itself and its own f32 roundings; all errors may have one sign:
    the tail's outputs by 2^-(32 - log2) of themselves."""
    n = 2
    c = Case([ctx], n, 2, 1, seed=11, chain=True, guard=3 if ctx > 2048 else 40)
    c.q[:], c.k[:] = 0, 0
    c.q[..., 0] = 1.0
    c.k[5, :, 0] = np.float16(log2 * np.log(2.0) * HD ** 0.5)
    c.v[:] = 2.0 ** (log2 - 14)
    c.v[5] = 0.0
    got = vals(_attend(ops, c.dev(), 2, 1))[0]
    w = np.exp(-float(c.k[5, 0, 0]) * HD ** -0.5)
    for i in range(n):
        tail = ctx + i  # rows that it sees but for row 5
        want = tail * w * 2.0 ** (log2 - 14) / (1 + tail * w)
        tol = 2.0 ** -11 + 2.0 ** -(32 - log2) * 1.5 + 2 * ctx * 2.0 ** -24 + 2.0 ** -18
        assert np.abs(got[i] / want - 1).max() <= tol
