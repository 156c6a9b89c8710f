"""Host-side tests of the serving nodes: what they refuse, and that a refused call has changed nothing."""
from __future__ import annotations

import numpy as np
import pytest

from modelsharp_amd import native, serving_kernels
from modelsharp_amd.graph import GraphContext, GraphNode, ModelSharpException
from modelsharp_amd.serving_kernels import HipLoraMatMulNBitsKernel, HipPagedAttentionKernel


@pytest.fixture
def on_the_host(monkeypatch):
    """The nodes on host tensors, with the names of the library's launches in the list returned."""
    import torch
    calls = []
    for name in ("paged_append", "paged_attention"):
        monkeypatch.setattr(native, name, lambda *a, n=name: calls.append(n))
    monkeypatch.setattr(serving_kernels, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, **k: t)
    return calls


def step(D, T=2, H=4, G=2, packed=True):
    """A PagedAttention node of one request of T tokens and its inputs."""
    import torch
    z = torch.zeros
    values = {"kc": z(4, 16, G, D), "vc": z(4, 16, G, D), "cu": np.array([0, T], np.int32), "past": np.array([3], np.int32),
              "table": np.array([[0, 1]], np.int32), "q": z(T, (H + (2 * G if packed else 0)) * D), "k": z(T, G * D),
              "v": z(T, G * D)}
    node = GraphNode("PagedAttention", "a", ["q", "" if packed else "k", "" if packed else "v", "kc", "vc", "cu", "past",
                                             "table"], ["o"], {"num_heads": H, "kv_num_heads": G})
    return node, GraphContext(values)


def run(node, ctx):
    k = HipPagedAttentionKernel()
    k._run(node, ctx)


def test_attention_takes_the_step(on_the_host):
    run(*step(64))
    assert on_the_host == ["paged_append", "paged_attention"]


@pytest.mark.parametrize("D,words", [(12, "multiple of 8"), (264, "multiple of 8")])
def test_what_attention_refuses_is_refused_before_the_append(on_the_host, D, words):
    with pytest.raises(native.HipError, match=words):
        run(*step(D))
    assert on_the_host == []


def test_descriptors_that_attention_refuses():
    d = dict(tokens=4, requests=2, num_heads=4, kv_num_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4,
             cache_type=native.MS_HIP_DTYPE_F16, local_window_size=-1)
    native.paged_attention_check(native.PagedDesc(**d))
    # a bound that is far too small splits the keys less rather than pass what a launch can have
    native.paged_attention_check(native.PagedDesc(**{**d, "tokens": 2 ** 21, "requests": 1, "max_new": 1, "num_pages": 2 ** 20,
                                                     "max_pages": 2 ** 20}))
    for kw, words in ((dict(head_dim=36), "multiple of 8"), (dict(num_heads=3), "multiple of kv_num_heads"),
                      (dict(tokens=2 ** 26, max_new=1, num_heads=8, kv_num_heads=8, head_dim=8), "too many workgroups")):
        with pytest.raises(native.HipError, match=words):
            native.paged_attention_check(native.PagedDesc(**{**d, **kw}))
    assert native.load().ms_hip_paged_attention_check(None) == native.MS_HIP_ERR_INVALID


@pytest.mark.parametrize("there", [1, 2], ids=["key", "value"])
def test_key_and_value_come_together(on_the_host, there):
    """One without the other is refused; it was read as a packed query."""
    node, ctx = step(64)
    node.inputs[there] = "kv"[there - 1]
    with pytest.raises(ModelSharpException, match="key and value must be given together"):
        run(node, ctx)
    assert on_the_host == []


@pytest.mark.parametrize("bad", [np.zeros((1, 2, 8), np.float64), np.zeros((2, 8), np.float16),
                                 np.zeros((1, 2, 8), np.int32)], ids=["f64", "2-D", "i32"])
def test_a_refused_adapter_initializer_is_refused_again(bad):
    """(It was kept before it was looked at: the second call took 64-bit weights as 32-bit ones.)"""
    import torch
    k = HipLoraMatMulNBitsKernel()
    ctx = GraphContext({"w": bad}, ["w"])
    for _ in range(3):
        with pytest.raises(ModelSharpException, match="3-D fp32 or fp16"):
            k._adapter(ctx, "w", torch.device("cpu"))
    assert not k._weights
    good = np.zeros((1, 2, 8), np.float16)
    ctx = GraphContext({"w": good}, ["w"])
    first = k._adapter(ctx, "w", torch.device("cpu"))
    assert k._adapter(ctx, "w", torch.device("cpu")).data_ptr() == first.data_ptr()   # uploaded once
