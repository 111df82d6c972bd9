"""Streams, scratch words and workspaces of another device are refused (runs without a GPU:
what is asked is the host's check, before any CUDA call)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

ONE = torch.device("cuda", 1)


class OnZero:
    """A tensor of cuda:0, as far as these checks look."""
    device = torch.device("cuda", 0)
    lengths = row_offset = k_pool = v_pool = None


def calls(ops, engine_mod):
    t = OnZero()
    return [
        lambda **kw: ops.attention_tree(t, t, t, t, t, t, t, 8, 2, **kw),
        lambda **kw: ops.kv_append_attention_tree(t, t, t, t, t, t, t, t, t, 8, 2, **kw),
        lambda **kw: ops.verify_tree(t, t, t, t, t, **kw),
        lambda **kw: ops.kv_commit([t], t, t, t, t, **kw),
    ]


@pytest.mark.parametrize("i", range(4))
def test_streams_of_another_device(ops, engine_mod, i):
    other = SimpleNamespace(cuda_stream=1234, device=ONE)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        calls(ops, engine_mod)[i](stream=other)


def test_streams_of_another_device_in_the_engine(ops, engine_mod):
    other = SimpleNamespace(cuda_stream=1234, device=ONE)
    layer = SimpleNamespace(lengths=OnZero(), device=OnZero.device)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        engine_mod.commit_layers([layer], OnZero(), OnZero(), stream=other)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        engine_mod.BatchedDecodeAttention.tree_step(layer, None, None, None, None, stream=other)


def test_an_engine_made_for_the_device_of_its_day(ops, engine_mod):
    """An engine made for "cuda" is on the device that was current then."""
    other = SimpleNamespace(cuda_stream=1234, device=ONE)
    layer = SimpleNamespace(lengths=OnZero(), device=torch.device("cuda"))
    with pytest.raises(ValueError, match="stream is on cuda:1, the tensors on cuda:0"):
        engine_mod.BatchedDecodeAttention.tree_step(layer, None, None, None, None, stream=other)


def test_the_output_is_where_the_queries_are(engine_mod, monkeypatch):
    """Not on the device that is current when the step runs (stand-ins: meta and cpu)."""
    seen = []
    monkeypatch.setattr(engine_mod.ops, "kv_append_attention_tree", lambda *a, **kw: seen.append(a[8]))
    names = "k_pool v_pool row_offset lengths heads kv_heads head_dim scale scratch region_rows"
    layer = SimpleNamespace(device=torch.device("cpu"), **{n: None for n in names.split()})
    q = torch.empty(1, 2, 8, 128, dtype=torch.float16, device="meta")
    out = engine_mod.BatchedDecodeAttention.tree_step(layer, q, None, None, None)
    assert out is seen[0] and out.device == q.device and out.shape == q.shape


@pytest.mark.parametrize("i", range(4))
def test_scratch_of_another_device(ops, engine_mod, i):
    scratch = SimpleNamespace(ptr=4096, nbytes=256, device=ONE)
    with pytest.raises(ValueError, match="scratch is on cuda:1"):
        calls(ops, engine_mod)[i](scratch=scratch)


@pytest.mark.parametrize("i", range(4))
def test_scratch_that_does_not_say_its_device(ops, engine_mod, i):
    """A decode workspace made for "cuda" serves as scratch: the call goes on to its tensors."""
    scratch = SimpleNamespace(ptr=4096, nbytes=256, device=torch.device("cuda"))
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        calls(ops, engine_mod)[i](scratch=scratch)


@pytest.mark.parametrize("i", range(2))
def test_workspace_of_another_device(ops, engine_mod, i):
    ws = SimpleNamespace(ptr=4096, nbytes=1 << 30, device=ONE)
    with pytest.raises(ValueError, match="workspace is on cuda:1"):
        calls(ops, engine_mod)[i](workspace=ws)
