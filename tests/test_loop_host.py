"""Host-side tests of what a server's loop needs around a step, and of attention behind shared prefixes: what the
entries refuse before anything is launched, the graph nodes' checks, and the plain forms the GPU tests use."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import loop_ref as ref
from modelsharp_amd import native
from modelsharp_amd.graph import GraphContext, GraphNode, KernelRegistry, ModelSharpException
from modelsharp_amd.serving_kernels import (HipPagedAttentionKernel, HipPagedStepCommitKernel, HipPagedStepPlanKernel,
                                            HipSampleTokensKernel, register_serving_kernels)

MB = 1 << 20   # addresses from here on are never followed: every call is refused or has nothing to do
F32, I32 = np.float32, np.int32


def refused(call, status, words):
    with pytest.raises(native.HipError, match=words) as e:
        call()
    assert e.value.status == status


def swapped(good, i, value):
    return [value if j == i else x for j, x in enumerate(good)]


def step(**kw):
    return native.StepDesc(**{**dict(tokens=6, requests=4, page_size=16, num_pages=20, max_pages=5), **kw})


PLAN = [(i + 1) * MB for i in range(10)]     # want, past, free, count | table, cu, used, requests, positions, slots
COMMIT = [(i + 1) * MB for i in range(8)]    # cu, used, done, keep | past, table, free, count


@pytest.mark.parametrize("kw,status,words", [
    (dict(tokens=-1), 1, "out of range"), (dict(tokens=2 ** 29 + 1), 1, "out of range"), (dict(requests=-1), 1, "negative"),
    (dict(max_pages=-1), 1, "negative"), (dict(page_size=0), 1, "page_size"), (dict(num_pages=0), 1, "num_pages"),
    (dict(num_pages=2 ** 28), 4, "rows"), (dict(requests=8193), 4, "8193 requests are more than 8192"),
    (dict(requests=8192, max_pages=2 ** 19), 4, "entries"),
])
def test_step_descriptor_refusals(kw, status, words):
    refused(lambda: native.step_check(step(**kw)), status, words)
    refused(lambda: native.paged_plan(step(**kw), *PLAN), status, words)
    refused(lambda: native.paged_commit(step(**kw), *COMMIT), status, words)


def test_step_descriptors_that_pass():
    for kw in (dict(), dict(tokens=0, requests=0, max_pages=0), dict(requests=8192), dict(tokens=2 ** 29),
               dict(page_size=1, num_pages=2 ** 31 - 1), dict(page_size=2 ** 31 - 1, num_pages=1)):
        native.step_check(step(**kw))


def test_null_descriptors():
    lib = native.load()
    for fn in (lib.ms_hip_step_check, lib.ms_hip_sample_check):
        assert fn(None) == native.MS_HIP_ERR_INVALID
    assert lib.ms_hip_sample_workspace_size(None) == 0
    d, s = paged(), native.SharedDesc(groups=1)
    for a, b in ((None, ctypes.byref(s)), (ctypes.byref(d), None), (None, None)):
        assert lib.ms_hip_paged_shared_attention_check(a, b) == native.MS_HIP_ERR_INVALID
        assert lib.ms_hip_paged_shared_attention_workspace_size(a, b) == 0
        assert lib.ms_hip_paged_shared_attention(a, b, *[MB] * 10, 0, None) == native.MS_HIP_ERR_INVALID
    assert lib.ms_hip_paged_plan(None, *PLAN, None) == native.MS_HIP_ERR_INVALID
    assert lib.ms_hip_paged_commit(None, *COMMIT, None) == native.MS_HIP_ERR_INVALID
    assert lib.ms_hip_sample(None, *[MB] * 9, 0, None) == native.MS_HIP_ERR_INVALID


def test_plan_buffers_are_checked():
    for i in range(10):
        refused(lambda: native.paged_plan(step(), *swapped(PLAN, i, None)), 1, "null")
        refused(lambda: native.paged_plan(step(), *swapped(PLAN, i, PLAN[i] + 2)), 1, "4-byte")
    sizes = (16, 16, 80, 4, 80, 20, 4, 24, 24, 24)
    for out in range(4, 10):   # each output on the last word of each other buffer
        for i in range(10):
            if i != out:
                refused(lambda: native.paged_plan(step(), *swapped(PLAN, out, PLAN[i] + sizes[i] - 4)), 1, "overlaps")
    refused(lambda: native.paged_plan(step(requests=0), *[None] * 2, *PLAN[2:4], None, None, *PLAN[6:]), 1, "null")   # cu


def test_commit_buffers_are_checked():
    for i in (0, 1, 4, 5, 6, 7):
        refused(lambda: native.paged_commit(step(), *swapped(COMMIT, i, None)), 1, "null")
    for i in range(8):
        refused(lambda: native.paged_commit(step(), *swapped(COMMIT, i, COMMIT[i] + 2)), 1, "4-byte")
    sizes = (20, 4, 16, 16, 16, 80, 80, 4)
    for out in range(4, 8):
        for i in range(8):
            if i != out:
                refused(lambda: native.paged_commit(step(), *swapped(COMMIT, out, COMMIT[i] + sizes[i] - 4)), 1, "overlaps")


# ---- sampling ------------------------------------------------------------------------------------

SAMPLE = [(i + 1) * 16 * MB for i in range(8)]   # logits, temperature, k, p, min_p, random | token, logprob
WS = 512 * MB


def sampled(**kw):
    return native.SampleDesc(**{**dict(rows=3, vocab=1000), **kw})


@pytest.mark.parametrize("kw,status,words", [
    (dict(rows=-1), 1, "rows"), (dict(vocab=0), 1, "vocab"), (dict(vocab=-5), 1, "vocab"), (dict(stride=999), 1, "stride"),
    (dict(stride=-1), 1, "stride"), (dict(vocab=2 ** 22 + 1), 4, "out of range"), (dict(rows=2 ** 31 - 1), 4, "out of range"),
])
def test_sample_descriptor_refusals(kw, status, words):
    refused(lambda: native.sample_check(sampled(**kw)), status, words)
    refused(lambda: native.sample(sampled(**kw), *SAMPLE, WS, 1 << 30), status, words)
    assert native.sample_workspace_size(sampled(**kw)) == 0


def test_sample_buffers_are_checked():
    n = native.sample_workspace_size(sampled())
    assert n > 0 and n % 16 == 0
    for i in (0, 5, 6):
        refused(lambda: native.sample(sampled(), *swapped(SAMPLE, i, None), WS, n), 1, "null")
    for i in range(8):
        refused(lambda: native.sample(sampled(), *swapped(SAMPLE, i, SAMPLE[i] + 2), WS, n), 1, "4-byte")
    for ws, size in ((None, n), (WS + 4, n), (WS, n - 1), (WS, 0), (WS, -1)):
        refused(lambda: native.sample(sampled(), *SAMPLE, ws, size), 1, "workspace of")
    sizes = (12000,) + (12,) * 7
    for i in range(8):   # each output on the last word of each other buffer, and the workspace on each
        for out in (6, 7):
            if i != out:
                refused(lambda: native.sample(sampled(), *swapped(SAMPLE, out, SAMPLE[i] + sizes[i] - 4), WS, n), 1, "overlaps")
        refused(lambda: native.sample(sampled(), *SAMPLE, SAMPLE[i] // 16 * 16, n), 1, "overlaps")
    # the last row ends with its width, not with its stride
    refused(lambda: native.sample(sampled(stride=2000), *swapped(SAMPLE, 6, SAMPLE[0] + 4 * (2 * 2000 + 999)), WS, n), 1,
            "overlaps")


def test_sample_workspace_is_bounded():
    """Rows are taken in batches: the workspace does not grow with them past 64 of them or 64 MB."""
    for vocab in (1, 1000, 32000, 151936, 2 ** 22):
        sizes = [native.sample_workspace_size(sampled(rows=r, vocab=vocab)) for r in (1, 64, 4096, 2 ** 20)]
        assert sizes == sorted(sizes) and 0 < sizes[0] and sizes[-1] <= max(64 * MB, 64 * sizes[0]) + 16


def test_calls_with_nothing_to_do():
    assert native.sample_workspace_size(sampled(rows=0)) == 0
    native.sample(sampled(rows=0), *[None] * 8)
    native.paged_shared_attention(paged(tokens=0), native.SharedDesc(groups=1), *[None] * 9)
    native.paged_shared_attention(paged(requests=0), native.SharedDesc(), *[None] * 9)


# ---- attention behind shared prefixes --------------------------------------------------------------

def paged(**kw):
    d = dict(tokens=4, requests=3, num_heads=4, kv_num_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4000,
             cache_type=native.MS_HIP_DTYPE_F16, local_window_size=-1)
    return native.PagedDesc(**{**d, **kw})


# q, cu, past, table, groups, shared, k, v, out
SHARED = [(i + 1) * 16 * MB for i in range(9)]


@pytest.mark.parametrize("kw,skw,status,words", [
    (dict(head_dim=12), {}, 4, "multiple of 8"), (dict(tokens=-1), {}, 1, "out of range"), (dict(cache_type=3), {}, 1, "fp32 or fp16"),
    ({}, dict(groups=-1), 1, "negative"), ({}, dict(max_shared=-1), 1, "negative"), ({}, dict(max_rest=-1), 1, "negative"),
    ({}, dict(groups=4), 1, "4 groups of 3 requests"), (dict(tokens=2 ** 26, num_heads=8, kv_num_heads=8, head_dim=8), {}, 4,
                                                        "too many workgroups"),
    # the merge of 2^26 rows in parts, where the parts themselves would do
    (dict(tokens=2 ** 20, num_heads=64, kv_num_heads=1, head_dim=8, max_pages=2 ** 16), {}, 4, "too many workgroups"),
])
def test_shared_descriptor_refusals(kw, skw, status, words):
    d, s = paged(**kw), native.SharedDesc(**{"groups": 1, **skw})
    refused(lambda: native.paged_shared_attention_check(d, s), status, words)
    refused(lambda: native.paged_shared_attention(d, s, *SHARED), status, words)
    assert native.paged_shared_attention_workspace_size(d, s) == 0


def test_shared_buffers_are_checked():
    d, s = paged(), native.SharedDesc(groups=2)
    n = native.paged_shared_attention_workspace_size(d, s)
    assert n > 0
    for i in range(9):
        refused(lambda: native.paged_shared_attention(d, s, *swapped(SHARED, i, None), WS, n), 1, "null")
    for i in (0, 1, 2, 3, 4, 5, 8):
        refused(lambda: native.paged_shared_attention(d, s, *swapped(SHARED, i, SHARED[i] + 2), WS, n), 1, "4-byte")
    for i in (6, 7):
        refused(lambda: native.paged_shared_attention(d, s, *swapped(SHARED, i, SHARED[i] + 8), WS, n), 1, "16-byte")
    for i in range(8):
        refused(lambda: native.paged_shared_attention(d, s, *swapped(SHARED, 8, SHARED[i]), WS, n), 1, "overlaps")
        refused(lambda: native.paged_shared_attention(d, s, *SHARED, SHARED[i], n), 1, "overlaps")
    refused(lambda: native.paged_shared_attention(d, s, *SHARED, SHARED[8], n), 1, "overlaps")
    refused(lambda: native.paged_shared_attention(d, s, *swapped(SHARED, 8, SHARED[4] + 8), WS, n), 1, "overlaps")


def test_what_shares():
    """16 MB of reading by the bounds, no window, groups; a workspace that serves the call alone as well."""
    def size(skw, **kw):
        return native.paged_shared_attention_workspace_size(paged(**kw), native.SharedDesc(**skw))

    alone = native.paged_attention_workspace_size(paged())
    shares = size(dict(groups=1))
    assert shares != alone
    assert size({}) == alone
    for skw, kw in ((dict(groups=1), dict(local_window_size=0)), (dict(groups=1, max_shared=100), {}), (dict(groups=3), {}),
                    (dict(groups=1), dict(max_total=500)), (dict(groups=1), dict(max_pages=100))):
        assert size(skw, **kw) == native.paged_attention_workspace_size(paged(**kw))
    # 2 requests more than groups, 512 bytes a position: 16384 positions
    at = [size(dict(groups=1, max_shared=p)) for p in (16383, 16384)]
    assert at[0] == alone and at[1] >= alone
    # 4 MB: alone, with nothing to merge
    native.paged_shared_attention_check(paged(tokens=2 ** 20, num_heads=64, kv_num_heads=1, head_dim=8), native.SharedDesc(groups=1))
    # bounds of any size
    big = 2 ** 31 - 1
    for kw in (dict(), dict(max_pages=big, max_total=big), dict(tokens=2 ** 20, requests=2 ** 20, max_pages=2 ** 20)):
        for skw in (dict(groups=1, max_shared=big, max_rest=big), dict(groups=3, max_shared=1, max_rest=1)):
            native.paged_shared_attention_check(paged(**kw), native.SharedDesc(**skw))


# ---- switches, nodes -----------------------------------------------------------------------------

def test_switches_cover_the_entries():
    lib = native.load()
    native.check(lib.ms_hip_debug_force_failure(1))
    try:
        for call in (lambda: native.paged_plan(step(), *PLAN), lambda: native.paged_commit(step(), *COMMIT),
                     lambda: native.sample(sampled(), *SAMPLE, WS, 1 << 30),
                     lambda: native.paged_shared_attention(paged(), native.SharedDesc(groups=1), *SHARED)):
            refused(call, native.MS_HIP_ERR_FORCED, "forced")
    finally:
        native.check(lib.ms_hip_debug_force_failure(0))


def test_registration():
    reg = register_serving_kernels(KernelRegistry())
    for op in ("PagedStepPlan", "PagedStepCommit", "SampleTokens"):
        assert reg.try_get(op)[0]


@pytest.fixture
def on_the_host(monkeypatch):
    """The nodes on host tensors; the names of the library's launches, with their descriptors, in the list returned."""
    import torch
    from modelsharp_amd import serving_kernels
    calls = []
    for name in ("paged_append", "paged_attention", "paged_shared_attention", "paged_plan", "paged_commit", "sample"):
        monkeypatch.setattr(native, name, lambda *a, n=name: calls.append((n, a)))
    monkeypatch.setattr(serving_kernels, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, **k: t)
    return calls


def pool(**kw):
    import torch
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    return {"table": z(4, 5), "past": z(4), "free": z(20), "count": z(1), "want": np.zeros(4, I32), "cu": z(5), "used": z(1),
            "done": np.zeros(4, I32), **kw}


def plan_node(**attrs):
    return GraphNode("PagedStepPlan", "p", ["table", "past", "free", "count", "want"], ["cu", "r", "p", "s", "used"],
                     {"tokens": 6, "block_size": 16, **attrs})


def test_plan_and_commit_nodes(on_the_host):
    ctx = GraphContext(pool())
    HipPagedStepPlanKernel()._run(plan_node(), ctx)
    assert [tuple(ctx.get_tensor(n).shape) for n in ("cu", "r", "p", "s", "used")] == [(5,), (6,), (6,), (6,), (1,)]
    node = GraphNode("PagedStepCommit", "c", ["table", "past", "free", "count", "cu", "used", "done"], ["t2", "p2"],
                     {"block_size": 16})
    HipPagedStepCommitKernel()._run(node, ctx)
    assert ctx.get_tensor("t2") is ctx.get_tensor("table") and ctx.get_tensor("p2") is ctx.get_tensor("past")
    (a, args), (b, brgs) = on_the_host
    assert (a, b) == ("paged_plan", "paged_commit") and brgs[4] is None   # no keep
    assert [getattr(args[0], f) for f, _ in args[0]._fields_] == [6, 4, 16, 20, 5]


@pytest.mark.parametrize("bad,words", [
    (dict(past=np.zeros(4, I32)), "int32 device tensor"), (dict(table=np.zeros((4, 5), I32)), "int32 device tensor"),
    (dict(free="f32"), "int32 device tensor"), (dict(table="strided"), "contiguous"), (dict(past="long"), "must be"),
    (dict(count="long"), "must be"), (dict(free="empty"), "must be"), (dict(want=np.zeros(3, I32)), "expected 4"),
], ids=str)
def test_refused_lists(on_the_host, bad, words):
    import torch
    make = {"f32": lambda: torch.zeros(20), "strided": lambda: torch.zeros(5, 4, dtype=torch.int32).T,
            "long": lambda: torch.zeros(3, dtype=torch.int32), "empty": lambda: torch.zeros(0, dtype=torch.int32)}
    ctx = GraphContext(pool(**{k: make[v]() if isinstance(v, str) else v for k, v in bad.items()}))
    with pytest.raises(ModelSharpException, match=words):
        HipPagedStepPlanKernel()._run(plan_node(), ctx)
    assert not on_the_host


def test_attributes_of_the_step_nodes(on_the_host):
    for attrs in (dict(tokens=-1), dict(block_size=0)):
        with pytest.raises(ModelSharpException, match="requires 'tokens'"):
            HipPagedStepPlanKernel().execute(plan_node(**attrs), GraphContext(pool()))
    with pytest.raises(native.HipError, match="page_size"):
        HipPagedStepCommitKernel()._run(GraphNode("PagedStepCommit", "c", ["table", "past", "free", "count", "cu", "used"], []),
                                        GraphContext(pool()))
    assert not on_the_host


def test_sample_node(on_the_host):
    import torch
    x, u = torch.zeros(2, 3, 50), np.zeros(6, F32)
    ctx = GraphContext({"x": x, "u": u, "t": np.ones(6, F32), "k": np.ones(6, np.int64), "short": u[:5]})

    def run(inputs, outputs=("y",)):
        HipSampleTokensKernel()._run(GraphNode("SampleTokens", "s", inputs, list(outputs)), ctx)

    run(["x", "u", "t", "k"], ("y", "lp"))
    assert tuple(ctx.get_tensor("y").shape) == tuple(ctx.get_tensor("lp").shape) == (2, 3)
    assert ctx.get_tensor("y").dtype == torch.int32
    run(["x", "u"])
    (_, full), (_, bare) = on_the_host
    assert full[4] is None and None not in full[1:4] and full[8] is not None   # no top_p; log-probabilities
    assert bare[2:6] == (None,) * 4 and bare[8] is None
    for inputs, words in ((["x"], "requires random"), (["x", "short"], "5 elements; expected 6"),
                          (["x", "u", "", "short"], "5 elements; expected 6")):
        with pytest.raises(ModelSharpException, match=words):
            run(inputs)
    assert len(on_the_host) == 2


def attention_node(values, groups=("g", "s")):
    import torch
    z = torch.zeros
    ctx = GraphContext({"kc": z(4, 16, 2, 64), "vc": z(4, 16, 2, 64), "q": z(6, 8 * 64), "table": np.zeros((4, 3), I32),
                        "cu": np.array([0, 1, 2, 4, 6], I32), "past": np.array([30, 33, 32, 5], I32), **values})
    return GraphNode("PagedAttention", "a", ["q", "", "", "kc", "vc", "cu", "past", "table", "", "", "", "", *groups], ["o"],
                     {"num_heads": 4, "kv_num_heads": 2}), ctx


def test_attention_node_takes_groups(on_the_host):
    node, ctx = attention_node({"g": np.array([0, 3], I32), "s": np.array([30], I32)})
    HipPagedAttentionKernel()._run(node, ctx)
    assert [n for n, _ in on_the_host] == ["paged_append", "paged_shared_attention"]
    s = on_the_host[1][1][1]
    assert (s.groups, s.max_shared, s.max_rest) == (1, 30, 7)   # the last request, in no group, has 7
    import torch
    node, ctx = attention_node({"g": torch.tensor([0, 3], dtype=torch.int32), "s": torch.tensor([30], dtype=torch.int32)})
    HipPagedAttentionKernel()._run(node, ctx)
    s = on_the_host[3][1][1]
    assert (s.groups, s.max_shared, s.max_rest) == (1, 0, 0)    # not fetched for it
    node, ctx = attention_node({"g": np.array([0], I32), "s": np.zeros(0, I32)})
    HipPagedAttentionKernel()._run(node, ctx)
    assert on_the_host[5][1][1].groups == 0


def test_attention_node_knows_lengths_of_zero(on_the_host):
    """The entry's 0 is "not known": host lengths that are all zero are a bound of 1, not of the table's width."""
    node, ctx = attention_node({"g": np.array([0, 2, 4], I32), "s": np.zeros(2, I32)})
    HipPagedAttentionKernel()._run(node, ctx)
    s = on_the_host[1][1][1]
    assert (s.groups, s.max_shared, s.max_rest) == (2, 1, 34)
    node, ctx = attention_node({"g": np.array([0, 4], I32), "s": np.array([48], I32), "past": np.full(4, 48, I32), "cu": np.zeros(5, I32)})
    HipPagedAttentionKernel()._run(node, ctx)
    s = on_the_host[3][1][1]
    assert (s.groups, s.max_shared, s.max_rest) == (1, 48, 1)


@pytest.mark.parametrize("values,groups,words", [
    (dict(g=np.array([0, 3], I32)), ("g",), "given together"), (dict(s=np.array([3], I32)), ("", "s"), "given together"),
    (dict(g=np.array([0, 3, 4], I32), s=np.array([3], I32)), ("g", "s"), "3 elements; expected 2"),
    (dict(g=np.arange(6, dtype=I32), s=np.zeros(5, I32)), ("g", "s"), "5 groups of 4 requests"),
])
def test_attention_node_refuses_before_the_append(on_the_host, values, groups, words):
    node, ctx = attention_node(values, groups)
    with pytest.raises((ModelSharpException, native.HipError), match=words):
        HipPagedAttentionKernel()._run(node, ctx)
    assert not on_the_host


# ---- the plain forms themselves ---------------------------------------------------------------------

def test_plain_plan_and_commit_by_hand():
    table = np.array([[3, -1, -1], [5, 6, -1], [-1, -1, -1]], I32)
    free = np.array([1, 2, 4, 0], I32)
    # 4 rows a page; request 0 has 3 cached and wants 2, request 1 has 8 and wants 1, request 2 wants 3
    cu, used, request, position, slot, t = ref.plan([2, 1, 3], [3, 8, 0], free, 3, table, 6, 4, 8)
    assert cu.tolist() == [0, 2, 3, 6] and used == 3
    assert t.tolist() == [[3, 4, -1], [5, 6, 2], [1, -1, -1]]
    assert request.tolist() == [0, 0, 1, 2, 2, 2] and position.tolist() == [3, 4, 8, 0, 1, 2]
    assert slot.tolist() == [15, 16, 8, 4, 5, 6]
    # one row less: the last waits, and one page less
    cu, used, request, *_ = ref.plan([2, 1, 3], [3, 8, 0], free, 3, table, 5, 4, 8)
    assert cu.tolist() == [0, 2, 3, 3] and used == 2 and request.tolist() == [0, 0, 1, -1, -1]
    assert ref.plan([2, 1, 3], [3, 8, 0], free, 2, table, 6, 4, 8)[0].tolist() == [0, 2, 3, 3]
    past, tt, f, n = ref.commit([0, 2, 3, 6], 3, [0, 1, 0], [0, 1, 0], [3, 8, 0], t, free, 3, 4, 8)
    assert past.tolist() == [5, 0, 3] and n == 2 and f[:2].tolist() == [6, 2]
    assert tt.tolist() == [[3, 4, -1], [5, -1, -1], [1, -1, -1]]


def test_plain_sampling_by_hand():
    row = np.log(np.array([4.0, 2.0, 1.0, 1.0], F32))
    for u, token in ((0.0, 0), (0.49, 0), (0.51, 1), (0.74, 1), (0.76, 2), (0.99, 3)):
        assert ref.sample(row, u=u)[0] == token
    assert ref.sample(row, k=2, u=0.9)[0] == 1 and np.isclose(ref.sample(row, k=2, u=0.9)[1], np.log(1 / 3))
    assert ref.sample(row, k=3, u=0.99)[0] == 2            # of equal ones the first
    assert ref.sample(row, p=0.6, u=0.99)[0] == 1 and ref.sample(row, p=0.4, u=0.99)[0] == 0
    assert ref.sample(row, m=0.3, u=0.99)[0] == 1 and ref.sample(row, t=0.0, u=0.99)[0] == 0
    assert np.isclose(ref.sample(row, t=0.5, u=0.0)[1], np.log(16 / 22))
    assert ref.sample(np.full(3, -np.inf))[0] == -1 and np.isnan(ref.sample(np.full(3, np.nan))[1])
    # (logs in 32 bits are off by 2^-25; equal logits have equal weights)
    assert ref.near_a_border(np.zeros(4, F32), u=0.5) and not ref.near_a_border(row, u=0.5)
