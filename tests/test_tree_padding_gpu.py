"""Padded batches: what stands behind tree_len is nobody's tree and no error."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_tree_gpu import HD, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctx,n,nh,nkv,tree_len", [
    ([150], 8, 40, 8, [5]),                      # a small pool, one CTA or a cluster per head
    ([60], 8, 8, 1, [0]),
    ([1900], 40, 2, 2, [33]),
    ([130, 0, 511, 96, 250], 32, 20, 4, [0, 1, 17, 31, 5]),
    ([700, 90, 30], 61, 40, 8, [1, 26, 60]),     # several tiles
])
def test_parents_of_absent_nodes(ops, ctx, n, nh, nkv, tree_len):
    c = Case(ctx, n, nh, nkv, seed=sum(tree_len), tree_len=tree_len)
    d = c.dev()
    for b, m in enumerate(tree_len):
        rest = torch.arange(n - m, dtype=torch.int32)
        d["parents"][b, m:] = torch.where(rest % 3 == 0, 2 ** 31 - 1 - rest, -9 - rest).cuda()
    for append in (False, True):
        sc = ops.Scratch()
        o = torch.full(d["q"].shape, 9.0, dtype=torch.float16, device="cuda")
        args = (d["row_offset"], d["seq_len"], d["parents"], o, nh, nkv, HD)
        if append:
            rows = [c.off[b] + c.ctx[b] + np.arange(n) for b in range(c.b)]
            new = [torch.from_numpy(np.stack([np.take(p, r, 0, mode="clip") for r in rows])).cuda()
                   for p in (c.k, c.v)]
            ops.kv_append_attention_tree(d["q"], *new, d["k_pool"], d["v_pool"], *args,
                                         tree_len=d["tree_len"], scratch=sc)
        else:
            ops.attention_tree(d["q"], d["k_pool"], d["v_pool"], *args, tree_len=d["tree_len"],
                               scratch=sc)
        c.check(o)
        assert sc.check() == 0


def test_parents_of_present_nodes_are_checked(ops):
    for ctx, n in (([40], 8), ([500, 40], 40)):
        m = [n - 2] * len(ctx)
        c = Case(ctx, n, 8, 2, seed=1, tree_len=m)
        d = c.dev()
        d["parents"][0, n - 3] = n
        c.parents[0, n - 3] = -1
        sc = ops.Scratch()
        o = torch.empty_like(d["q"])
        ops.attention_tree(d["q"], d["k_pool"], d["v_pool"], d["row_offset"], d["seq_len"],
                           d["parents"], o, 8, 2, HD, tree_len=d["tree_len"], scratch=sc)
        c.check(o)
        assert sc.check() == 4
