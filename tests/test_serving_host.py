"""Host-side tests of the serving-step operators that need no GPU: what the entries refuse before
anything is launched, the graph nodes' checks, and the plain 64-bit forms the GPU tests use."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import serving_ref as ref
from modelsharp_amd import native
from modelsharp_amd.graph import GraphContext, GraphNode, KernelRegistry, ModelSharpException
from modelsharp_amd.serving_kernels import (HipLoraMatMulNBitsKernel, HipPagedAttentionKernel, HipQkNormRotaryKernel,
                                            register_serving_kernels)

P = 1 << 20   # an address that is never followed: every call here is refused or has nothing to do


def paged(**kw):
    d = dict(tokens=4, requests=2, num_heads=4, kv_num_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4,
             cache_type=native.MS_HIP_DTYPE_F16, local_window_size=-1)
    return native.PagedDesc(**{**d, **kw})


def refused(call, status, words):
    with pytest.raises(native.HipError, match=words) as e:
        call()
    assert e.value.status == status


@pytest.mark.parametrize("kw,status,words", [
    (dict(num_heads=0), 1, "positive 'num_heads'"), (dict(kv_num_heads=-1), 1, "positive 'num_heads'"),
    (dict(num_heads=70000, kv_num_heads=2), 1, "65535"), (dict(num_heads=5), 1, "must be a multiple of kv_num_heads=2"),
    (dict(head_dim=0), 1, "head_dim"), (dict(head_dim=1032), 1, "head_dim"), (dict(tokens=-1), 1, "out of range"),
    (dict(tokens=2 ** 30), 1, "out of range"), (dict(requests=-1), 1, "negative"), (dict(max_new=-1), 1, "negative"),
    (dict(max_total=-1), 1, "negative"), (dict(max_pages=-1), 1, "negative"), (dict(page_size=0), 1, "page_size"),
    (dict(num_pages=0), 1, "num_pages"), (dict(num_pages=2 ** 28), 4, "rows"), (dict(cache_type=3), 1, "fp32 or fp16"),
    (dict(q_stride=255), 1, "stride"), (dict(k_stride=-4), 1, "stride"), (dict(v_stride=127), 1, "stride"),
    (dict(do_rotary=1, cos_rows=0, cos_cols=32), 1, "cos_cache"), (dict(do_rotary=1, cos_rows=9), 1, "cos_cache"),
])
def test_paged_descriptor_refusals(kw, status, words):
    d = paged(**kw)
    refused(lambda: native.check(native.load().ms_hip_paged_check(ctypes.byref(d))), status, words)
    refused(lambda: native.paged_append(d, P, P, P, None, None, P, P, P, P, P, P, P, P), status, words)
    refused(lambda: native.paged_attention(d, P, P, P, P, P, P, P), status, words)
    assert native.paged_attention_workspace_size(d) == 0


def test_null_descriptors_are_refused():
    lib = native.load()
    for fn in (lib.ms_hip_paged_check, lib.ms_hip_qk_norm_check, lib.ms_hip_lora_check):
        assert fn(None) == native.MS_HIP_ERR_INVALID
    assert lib.ms_hip_paged_attention_workspace_size(None) == 0 and lib.ms_hip_lora_workspace_size(None) == 0


def test_paged_buffers_are_checked():
    MB = 1 << 20
    q, k, v, cu, past, table, out, kc, vc = (P + i * MB for i in range(9))
    good = [q, k, v, None, None, cu, past, table, None, None, out, kc, vc]
    for i in (0, 1, 2, 5, 6, 7, 10, 11, 12):   # null
        refused(lambda: native.paged_append(paged(), *[None if j == i else x for j, x in enumerate(good)]), 1, "null")
    for i in (0, 1, 2, 5, 6, 7, 10):
        refused(lambda: native.paged_append(paged(), *[x + 2 if j == i else x for j, x in enumerate(good)]), 1, "4-byte")
    for i in (11, 12):
        refused(lambda: native.paged_append(paged(), *[x + 8 if j == i else x for j, x in enumerate(good)]), 1, "16-byte")
    for i, other in ((10, q + 16), (10, k), (10, v), (10, kc), (11, vc), (12, q), (11, k)):   # overlaps
        refused(lambda: native.paged_append(paged(), *[other if j == i else x for j, x in enumerate(good)]), 1, "overlaps")
    # in place only where the rows lie back to back
    refused(lambda: native.paged_append(paged(q_stride=512), q, k, v, None, None, cu, past, table, None, None, q, kc, vc), 1,
            "overlaps")
    refused(lambda: native.paged_append(paged(do_rotary=1, cos_rows=8, cos_cols=32), *good), 1, "cos_cache")
    att = [q, cu, past, table, kc, vc, out]
    for i in range(7):
        refused(lambda: native.paged_attention(paged(), *[None if j == i else x for j, x in enumerate(att)]), 1, "null")
    for i in (0, 1, 2, 3, 6):
        refused(lambda: native.paged_attention(paged(), *[x + 1 if j == i else x for j, x in enumerate(att)]), 1, "4-byte")
    for i in (4, 5):
        refused(lambda: native.paged_attention(paged(), *[x + 4 if j == i else x for j, x in enumerate(att)]), 1, "16-byte")
    for other in (q, q + 1024, kc, vc):
        refused(lambda: native.paged_attention(paged(), *att[:6], other), 1, "overlaps")
    d = paged()
    n = native.paged_attention_workspace_size(d)
    if n:
        refused(lambda: native.paged_attention(d, *att, out, n), 1, "overlaps")
    for D in (4, 63, 264, 512):   # append takes them, attention does not
        refused(lambda: native.paged_attention(paged(head_dim=D), *att), 4, "multiple of 8 up to 256")


def test_empty_calls_launch_nothing():
    for kw in (dict(tokens=0), dict(requests=0)):
        native.paged_append(paged(**kw), None, None, None, None, None, None, None, None, None, None, None, None, None)
        native.paged_attention(paged(**kw), None, None, None, None, None, None, None)
    native.qk_norm_rotary(native.QkNormDesc(tokens=0, num_heads=1, kv_num_heads=1, head_dim=8), *[None] * 9)
    native.lora(native.LoraDesc(tokens=0, K=8, N=8, adapters=1, max_rank=1, weight_type=1), *[None] * 9, 0)


def test_qk_norm_refusals():
    MB = 1 << 20
    q, k, pos, cos, sin, qo, ko = (P + i * MB for i in range(7))

    def d(**kw):
        return native.QkNormDesc(**{**dict(tokens=4, num_heads=4, kv_num_heads=2, head_dim=64, do_rotary=1, cos_rows=8,
                                           cos_cols=32), **kw})

    for kw, words in ((dict(num_heads=3), "multiple"), (dict(tokens=-2), "range"), (dict(head_dim=2000), "head_dim"),
                      (dict(q_stride=8), "stride"), (dict(k_stride=100), "stride"), (dict(cos_rows=0), "cos_cache")):
        refused(lambda: native.qk_norm_rotary(d(**kw), q, k, None, None, pos, cos, sin, qo, ko), 1, words)
    good = [q, k, None, None, pos, cos, sin, qo, ko]
    for i, words in ((0, "null"), (1, "null"), (7, "null"), (8, "null"), (4, "positions"), (5, "cos_cache"), (6, "sin_cache")):
        refused(lambda: native.qk_norm_rotary(d(), *[None if j == i else x for j, x in enumerate(good)]), 1, words)
    for i, other in ((7, k), (8, q), (7, ko), (7, q + 4), (8, k + 4)):
        refused(lambda: native.qk_norm_rotary(d(), *[other if j == i else x for j, x in enumerate(good)]), 1, "overlaps")
    refused(lambda: native.qk_norm_rotary(d(q_stride=300), q, k, None, None, pos, cos, sin, q, ko), 1, "overlaps")


def test_lora_refusals():
    MB = 1 << 20
    x, a, b, ranks, scales, which, base, y, ws = (P + i * MB for i in range(9))

    def d(**kw):
        return native.LoraDesc(**{**dict(tokens=4, K=64, N=32, adapters=2, max_rank=8,
                                         weight_type=native.MS_HIP_DTYPE_F16), **kw})

    good = [x, a, b, ranks, scales, which, base, y, ws]
    n = native.lora_workspace_size(d())
    assert n >= 4 * 16 * 4
    for kw, status in ((dict(tokens=-1), 1), (dict(K=0), 1), (dict(N=0), 1), (dict(adapters=0), 1), (dict(max_rank=0), 1),
                       (dict(max_rank=1025), 4), (dict(weight_type=0), 1), (dict(tokens=2 ** 25), 4)):
        refused(lambda: native.lora(d(**kw), *good, n), status, "lora")
        assert native.lora_workspace_size(d(**kw)) == 0
    for i in (0, 1, 2, 5, 7):
        refused(lambda: native.lora(d(), *[None if j == i else v for j, v in enumerate(good)], n), 1, "null")
    for i in (0, 3, 4, 5, 6, 7):
        refused(lambda: native.lora(d(), *[v + 2 if j == i else v for j, v in enumerate(good)], n), 1, "4-byte")
    for i in (1, 2):
        refused(lambda: native.lora(d(), *[v + 1 if j == i else v for j, v in enumerate(good)], n), 1, "aligned to their type")
    refused(lambda: native.lora(d(), *good, n - 1), 1, "workspace of")
    refused(lambda: native.lora(d(), *good[:-1], None, n), 1, "workspace of")
    refused(lambda: native.lora(d(), *good[:-1], ws + 4, n), 1, "workspace of")
    for i, other in ((7, x), (7, a), (7, b), (7, base + 4)):
        refused(lambda: native.lora(d(), *[other if j == i else v for j, v in enumerate(good)], n), 1, "overlaps")
    for other in (x, base, y):
        refused(lambda: native.lora(d(), *good[:-1], other, n), 1, "workspace overlaps")


def test_switches_cover_the_serving_entries():
    lib = native.load()
    native.check(lib.ms_hip_debug_force_failure(1))
    try:
        refused(lambda: native.paged_append(paged(), *[P] * 13), native.MS_HIP_ERR_FORCED, "forced")
        refused(lambda: native.paged_attention(paged(), *[P] * 7), native.MS_HIP_ERR_FORCED, "forced")
        refused(lambda: native.qk_norm_rotary(native.QkNormDesc(tokens=1, num_heads=1, kv_num_heads=1, head_dim=8),
                                              *[P] * 9), native.MS_HIP_ERR_FORCED, "forced")
        refused(lambda: native.lora(native.LoraDesc(tokens=1, K=8, N=8, adapters=1, max_rank=1, weight_type=1), *[P] * 9, 0),
                native.MS_HIP_ERR_FORCED, "forced")
    finally:
        native.check(lib.ms_hip_debug_force_failure(0))


def test_registration_and_node_checks():
    reg = register_serving_kernels(KernelRegistry())
    for op in ("PagedAttention", "QkNormRotary", "LoraMatMulNBits"):
        assert reg.try_get(op)[0]
    k = HipPagedAttentionKernel()
    node = GraphNode("PagedAttention", "a", ["q"] + [""] * 7, ["o"], {"num_heads": 3, "kv_num_heads": 2})
    with pytest.raises(ModelSharpException, match="multiple of kv_num_heads=2"):
        k.execute(node, GraphContext({}))
    node.attributes = {"num_heads": 4, "kv_num_heads": 2, "softcap": 30.0}
    with pytest.raises(ModelSharpException, match="softcap"):
        k.execute(node, GraphContext({}))
    with pytest.raises(ModelSharpException, match="positive 'num_heads'"):
        HipQkNormRotaryKernel().execute(GraphNode("QkNormRotary", "r", ["q", "k"], ["a", "b"]), GraphContext({}))


def test_nodes_take_their_inputs_to_the_first_ones_device():
    """A tensor on another device, the host among them, never reaches a kernel by its address."""
    import torch
    x = torch.zeros(2, 64)
    for k, node in (
            (HipPagedAttentionKernel(), GraphNode("PagedAttention", "a", ["x"] + [""] * 7, ["o"],
                                                  {"num_heads": 1, "kv_num_heads": 1})),
            (HipQkNormRotaryKernel(), GraphNode("QkNormRotary", "r", ["x", "x"], ["a", "b"],
                                                {"num_heads": 1, "kv_num_heads": 1})),
            (HipLoraMatMulNBitsKernel(), GraphNode("LoraMatMulNBits", "l", ["x"] * 9, ["o"], {}))):
        with pytest.raises(ModelSharpException, match="is a tensor on cpu"):
            k.execute(node, GraphContext({"x": x}))
    meta = torch.device("meta")
    ctx = GraphContext({"g": torch.ones(8), "c": torch.ones(4, 4), "a": torch.zeros(1, 2, 8), "n": torch.zeros(3)})
    k = HipLoraMatMulNBitsKernel()
    assert k._gamma(ctx, "g", 8, meta).device == meta
    assert all(t.device == meta for t in k._rotary(GraphNode("", "", ["c", "c"], []), ctx, 0, meta))
    assert k._adapter(ctx, "a", meta).device == meta and k._lengths(ctx, "n", 3, meta).device == meta
    w = np.zeros((1, 2, 8), np.float16)   # an initializer, kept from its first use on another device
    k._weights[id(w)] = (w, torch.zeros(1, 2, 8, dtype=torch.float16))
    assert k._adapter(GraphContext({"w": w}, ["w"]), "w", meta).device == meta


# ---- the plain forms themselves ---------------------------------------------------------------------

def test_plain_attention_against_a_hand_worked_case():
    b = ref.Batch(0, [2], [1], 1, 8, 2, np.float32)
    b.k[:], b.v[:] = 0.0, 0.0
    for j in range(3):
        b.v.reshape(-1, 1, 8)[b.row(0, j)] = j + 1.0
    q = np.zeros((2, 8), np.float32)
    out, _, longest = ref.attention(b, q, 1)          # equal scores: means of 1, 2 and of 1, 2, 3
    assert longest == 3 and np.allclose(out[0], 1.5) and np.allclose(out[1], 2.0)
    out, _, _ = ref.attention(b, q, 1, window=1)      # only the token itself
    assert np.allclose(out[0], 2.0) and np.allclose(out[1], 3.0)
    assert (ref.attention(b, q, 1, window=0)[0] == 0).all()
    b.table[0, 0] = -1                                # positions 0 and 1 have no page
    out, _, _ = ref.attention(b, q, 1)
    assert (out[0] == 0).all() and np.allclose(out[1], 3.0)


def test_plain_norm_and_rotation():
    x = np.array([[3.0, 4.0, 0.0, 0.0]])
    n = ref.normed_rotated(x, np.ones(4), 0, None, None, False, 0.0)
    assert np.allclose(n, x / 2.5)
    cos, sin = np.zeros((2, 2)), np.ones((2, 2))      # a quarter turn
    assert np.allclose(ref.normed_rotated(x, None, 9, cos, sin, False, 0.0), [[0.0, 0.0, 3.0, 4.0]])
    assert np.allclose(ref.normed_rotated(x, None, 0, cos, sin, True, 0.0), [[-4.0, 3.0, 0.0, 0.0]])


def test_plain_lora():
    x = np.array([[1.0, 2.0], [1.0, 2.0], [5.0, 5.0]])
    a = np.array([[[1.0, 1.0], [9.0, 9.0]]])
    b = np.array([[[2.0, 9.0]]])
    y, _ = ref.lora(x, a, b, np.array([1]), np.array([0.5]), np.array([0, -1, 7]), np.ones((3, 1)))
    assert np.allclose(y[:, 0], [1 + 0.5 * 2 * 3, 1, 1])
