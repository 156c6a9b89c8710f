"""Attention behind prefixes that groups of requests share, on the GPU against the plain 64-bit form, which knows
nothing of groups."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from modelsharp_amd import native
from test_gpu_serving import check_attention, desc_of, dev, log, ptr, run_attention, stream

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32


WORTH = 16 << 20   # bytes that a call has to leave out, by its bounds, to share anything


def batch(seed, groups, G, D, page, dtype, spare_rows=0, extra_columns=0, roomy=True):
    """(batch, bounds, shared) of groups [(shared positions, [(new, own cached), ...]), ...]. Whole pages of a prefix
    are the same pages; a part of one is a copy in each request's own. A group of shared 0 shares nothing. A roomy
    batch's table is wide enough that a call without other bounds shares."""
    news = [n for _, members in groups for n, _ in members]
    pasts = [s + o for s, members in groups for _, o in members]
    if roomy:
        saved = max(1, len(news) - len(groups)) * page * 2 * G * D * np.dtype(dtype).itemsize   # by a page's positions
        extra_columns += -(-WORTH // saved)
    b = ref.Batch(seed, news, pasts, G, D, page, dtype, spare_rows=spare_rows, extra_columns=extra_columns)
    bounds, r = [0], 0
    for shared, members in groups:
        first = r
        for _ in members:
            whole, part = divmod(shared, page)
            b.table[r, :whole] = b.table[first, :whole]
            if part and r != first:
                for c in (b.k, b.v):
                    c[b.table[r, whole], :part] = c[b.table[first, whole], :part]
            r += 1
        bounds.append(r)
    return b, np.array(bounds, I32), np.array([s for s, _ in groups], I32)


def run_shared(b, bounds, shared, q, H, window=-1, scale=0.0, workspace=True, hints=False, stride=0, out=None):
    """paged_shared_attention's output, by the table's width or with exact bounds (hints); the call is one that
    shares but where the test says otherwise."""
    import torch
    d = desc_of(b, H, local_window_size=window, scale=scale, q_stride=stride)
    s = native.SharedDesc(groups=len(shared))
    if hints:
        total = np.add(b.news, b.pasts)
        d.max_new, d.max_total = max(b.news), int(total.max())
        mine = np.zeros(len(total), int)
        for g in range(len(shared)):
            mine[max(bounds[g], 0):max(bounds[g + 1], 0)] = shared[g]
        s.max_shared, s.max_rest = max(0, int(max(shared, default=0))), max(0, int((total - mine).max()))
    if workspace and 0 < len(shared) < len(b.news):
        prefix = s.max_shared or b.max_pages * b.page
        assert (len(b.news) - len(shared)) * prefix * 2 * b.G * b.D * b.k.itemsize >= WORTH
    o = torch.full((b.tokens, H * b.D), float("nan"), device="cuda") if out is None else dev(out)
    n = native.paged_shared_attention_workspace_size(d, s) if workspace else 0
    ws = torch.full((n // 4 + 64,), float("nan"), device="cuda")
    bufs = [dev(x) for x in (q, b.cu, b.past, b.table, bounds, shared, b.k, b.v)]
    native.paged_shared_attention(d, s, *map(ptr, bufs), ptr(o), ptr(ws) if n else None, n, stream())
    torch.cuda.synchronize()
    assert torch.isnan(ws[n // 4:]).all()   # nothing past the workspace
    return o.cpu().numpy()


def queries(b, H):
    return b.rng.standard_normal((b.tokens, H * b.D)).astype(F32) * F32(1.5)


# groups, H, G, D, page
CASES = [
    ([(1, [(1, 0)])], 1, 1, 8, 1),                                             # one request, one key behind one
    ([(16, [(1, 0), (1, 3)])], 14, 2, 64, 16),
    ([(700, [(1, 5), (1, 60), (1, 0), (1, 33)])], 14, 2, 64, 16),
    ([(333, [(1, i % 40) for i in range(70)])], 28, 4, 128, 16),               # more requests than lanes, a part of a page
    ([(48, [(1, 2)] * 3), (0, [(1, 9), (2, 100)]), (130, [(1, 7)] * 20)], 8, 8, 128, 10),
    ([(0, [(1, 30)]), (64, [(0, 5), (3, 0), (0, 0), (1, 70)]), (0, [(0, 4)])], 4, 2, 64, 16),   # without new tokens
    ([(500, [(17, 0), (33, 40)])], 6, 2, 96, 16),
    ([(90, [(64, 0), (1, 20), (100, 31)]), (200, [(5, 0)] * 4)], 28, 4, 128, 32),
    ([(1000, [(3, 2)] * 9)], 4, 4, 256, 16),
    ([(75, [(20, 3)] * 3)], 8, 2, 80, 7),
    ([(2050, [(1, i) for i in range(20)])], 16, 1, 128, 64),
    ([(40, [(2, 1)] * 2)] * 70, 2, 1, 64, 8),                                  # more groups than lanes
    ([(300, [(1, 3)] * 33), (299, [(1, 3)] * 2), (301, [(40, 0)])], 8, 2, 40, 24),
    ([(4100, [(1, 10)] * 5)], 32, 8, 128, 128),
]


@pytest.mark.parametrize("workspace", [True, False], ids=["shared", "alone"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_shared_attention(gpu, case, dtype, workspace):
    groups, H, G, D, page = CASES[case]
    log(f"shared {case} {dtype.__name__} workspace={workspace}")
    b, bounds, shared = batch(2000 + case, groups, G, D, page, dtype, spare_rows=3 * (case % 2), extra_columns=case % 3)
    q = queries(b, H)
    check_attention(run_shared(b, bounds, shared, q, H, workspace=workspace), b, q, H)


# with bounds as they are: groups, H, G, D, page
LARGE = [
    ([(2100, [(1, 3)] * 3)], 8, 8, 128, 16),
    ([(1100, [(1, i) for i in range(32)])], 28, 4, 128, 16),
    ([(3001, [(40, 7)] * 8)], 14, 2, 128, 16),
    ([(900, [(1, 5)] * 20), (1200, [(2, 0)] * 15)], 16, 2, 256, 24),
    ([(1000, [(1, 9)] * 16), (0, [(1, 30)] * 4), (1500, [(100, 3), (1, 0)])], 8, 4, 64, 32),
    ([(4005, [(1, 2)] * 40)], 4, 4, 40, 10),
    ([(640, [(3, 90)] * 33)], 12, 4, 96, 16),
    ([(3000, [(1, 400)] * 24)], 32, 1, 64, 64),
]


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_shared_attention_by_its_bounds(gpu, case, dtype):
    groups, H, G, D, page = LARGE[case]
    log(f"large {case} {dtype.__name__}")
    b, bounds, shared = batch(2100 + case, groups, G, D, page, dtype, spare_rows=2 * (case % 2), roomy=False)
    q = queries(b, H)
    check_attention(run_shared(b, bounds, shared, q, H, hints=True), b, q, H)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_bounds_that_are_too_small(gpu, dtype):
    """They choose the launch alone."""
    import torch
    groups, H, G, D, page = LARGE[4]
    b, bounds, shared = batch(9, groups, G, D, page, dtype)
    q = queries(b, H)
    bufs = [dev(x) for x in (q, b.cu, b.past, b.table, bounds, shared, b.k, b.v)]
    for new, total, prefix, rest in ((1, 0, 0, 1), (1, 0, 1500, 1), (2, 0, 900, 2), (0, 950, 900, 1)):
        d = desc_of(b, H, max_new=new, max_total=total)
        s = native.SharedDesc(groups=len(shared), max_shared=prefix, max_rest=rest)
        n = native.paged_shared_attention_workspace_size(d, s)
        out, ws = torch.full((b.tokens, H * D), float("nan"), device="cuda"), torch.empty(n // 4 + 4, device="cuda")
        log(f"bounds {new} {total} {prefix} {rest}")
        native.paged_shared_attention(d, s, *map(ptr, bufs), ptr(out), ptr(ws), n, stream())
        check_attention(out.cpu().numpy(), b, q, H)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_bounds_of_new_tokens_that_are_too_small_beside_large_tiles(gpu, dtype):
    """The prefix in tiles of 128 rows, the requests' own keys in tiles of 16 by a bound of few new tokens, and requests
    of more: every row has its own keys' records."""
    import torch
    H, G, D, prefix = 8, 2, 64, 5000
    b, bounds, shared = batch(11, [(prefix, [(40, 30)] * 6 + [(1, 500), (64, 0)])], G, D, 16, dtype, roomy=False)
    q = queries(b, H)
    rows, cus = b.tokens * H // G, torch.cuda.get_device_properties(0).multi_processor_count
    pad = lambda n: -(-rows // n) * n   # noqa: E731
    bufs = [dev(x) for x in (q, b.cu, b.past, b.table, bounds, shared, b.k, b.v)]
    for new in (1, 9, 16):
        d = desc_of(b, H, max_new=new)
        s = native.SharedDesc(groups=1, max_shared=prefix, max_rest=600)
        assert (len(b.news) - 1) * prefix * 2 * G * D * b.k.itemsize >= WORTH
        # what the launch goes by: few rows to a request, so many to the prefix that tiles of 128 take it
        assert new * H // G <= 64 < 40 * H // G and pad(128) * prefix * G / 2400 + 5 * cus < pad(16) * prefix * G / 1700
        n = native.paged_shared_attention_workspace_size(d, s)
        assert n > 2 * b.tokens * H * (D + 2) * 4   # shared, in several records
        out, ws = (torch.full((m,), float("nan"), device="cuda") for m in (b.tokens * H * D, n // 4 + 4))
        log(f"bound of {new} beside tiles of 128 rows, {dtype.__name__}")
        native.paged_shared_attention(d, s, *map(ptr, bufs), ptr(out), ptr(ws), n, stream())
        check_attention(out.reshape(b.tokens, -1).cpu().numpy(), b, q, H)


@pytest.mark.parametrize("new", [1, 40], ids=["tokens", "chunks"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_a_prefix_is_read_from_its_first_request(gpu, dtype, new):
    """The others' entries of the table for it are not looked at, which shows that it is shared."""
    H, G, D, page = 8, 2, 64, 16
    b, bounds, shared = batch(10, [(100, [(new, 30)] * 5), (64, [(new, 0)] * 2)], G, D, page, dtype)
    q = queries(b, H)
    want, mass, longest = ref.attention(b, q, H)
    tol = ref.attention_tolerance(mass, longest, D, float(np.abs(b.v).max()))
    bad = b.num_pages - 1 if b.num_pages - 1 not in b.table else int(np.setdiff1d(np.arange(b.num_pages), b.table)[0])
    b.k[bad], b.v[bad] = np.nan, np.nan
    log(f"first request {dtype.__name__} {new}")
    b.table[1:5, :6], b.table[6, :4] = bad, -1
    got = run_shared(b, bounds, shared, q, H)
    assert np.abs(got - want).max() <= tol
    assert np.isnan(run_shared(b, bounds, shared, q, H, workspace=False)).any()


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_requests_outside_the_groups(gpu, dtype):
    """Before the first group and behind the last; no group at all."""
    groups = [(0, [(1, 40), (2, 5)]), (160, [(1, 6)] * 7), (0, [(30, 100), (1, 3)])]
    b, bounds, shared = batch(1, groups, 2, 64, 16, dtype)
    q = queries(b, 8)
    log(f"outside {dtype.__name__}")
    check_attention(run_shared(b, bounds[1:3], shared[1:2], q, 8), b, q, 8)
    check_attention(run_shared(b, bounds[:1], shared[:0], q, 8), b, q, 8)
    assert np.array_equal(run_shared(b, bounds[:1], shared[:0], q, 8), run_attention(b, q, 8, hints=False))


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_a_window_shares_nothing(gpu, dtype):
    b, bounds, shared = batch(2, [(200, [(1, 6), (20, 3)] * 3)], 2, 128, 16, dtype)
    q = queries(b, 4)
    log(f"window {dtype.__name__}")
    for window in (0, 1, 50, 1000):
        assert np.array_equal(run_shared(b, bounds, shared, q, 4, window), run_attention(b, q, 4, window, hints=False))
    check_attention(run_shared(b, bounds, shared, q, 4, 50), b, q, 4, 50)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_shared_packed_rows_and_scale(gpu, dtype):
    H, G, D = 6, 2, 64
    b, bounds, shared = batch(3, [(100, [(4, 3), (1, 0), (40, 2)])], G, D, 16, dtype)
    packed = b.rng.standard_normal((b.tokens, (H + 2 * G) * D)).astype(F32)
    q = np.ascontiguousarray(packed[:, :H * D])
    log(f"packed {dtype.__name__}")
    for scale in (0.31, -0.2):
        check_attention(run_shared(b, bounds, shared, packed, H, scale=scale, stride=(H + 2 * G) * D), b, q, H, scale=scale)


@pytest.mark.parametrize("new", [1, 40], ids=["tokens", "chunks"])
@pytest.mark.parametrize("where,value", [("k", np.inf), ("k", -np.inf), ("k", np.nan), ("v", np.inf), ("v", np.nan), ("q", np.nan),
                                         ("k", 6e4), ("v", 6e4)])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_odd_values_behind_and_in_a_prefix(gpu, dtype, where, value, new):
    """One in the prefix reaches every row of its group, one in a request's own keys that request alone."""
    H, G, D = 4, 2, 64
    groups = [(120, [(new, 30), (new, 4)]), (50, [(new, 9)] * 2)]
    log(f"odd {where}={value} {dtype.__name__} {new}")
    for place in ((0, 70), (1, 121), (2, 49)):   # request, position
        b, bounds, shared = batch(4, groups, G, D, 16, dtype)
        q = queries(b, H)
        if where == "q":
            q[int(b.cu[place[0]]), 5] = value
        else:
            (b.k if where == "k" else b.v).reshape(-1, G, D)[b.row(*place), 1, 3] = value
            if place == (2, 49):   # a copy of the prefix's last, partial page
                (b.k if where == "k" else b.v).reshape(-1, G, D)[b.row(3, 49), 1, 3] = value
        check_attention(run_shared(b, bounds, shared, q, H), b, q, H)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_what_a_prefix_does_not_hold(gpu, dtype):
    """NaN and infinities in pages of nobody and in rows behind each request's last; a page of the prefix that is gone."""
    H, G, D = 8, 2, 128
    for new in (1, 50):
        b, bounds, shared = batch(5, [(100, [(new, 37), (new, 0), (new, 12)]), (33, [(new, 2)])], G, D, 16, dtype)
        q = queries(b, H)
        used = {b.row(r, j) for r in range(4) for j in range(b.pasts[r] + b.news[r])}
        free = np.setdiff1d(np.arange(b.num_pages * b.page), np.array(sorted(used)))
        k, v = b.k.reshape(-1, G, D), b.v.reshape(-1, G, D)
        k[free[::2]], v[free[::2]], k[free[1::2]], v[free[1::2]] = np.nan, np.nan, np.inf, -np.inf
        log(f"unseen {dtype.__name__} {new}")
        got = run_shared(b, bounds, shared, q, H)
        assert np.isfinite(got).all()
        check_attention(got, b, q, H, v_max=5.0)
        b.table[:3, 2] = -1
        check_attention(run_shared(b, bounds, shared, q, H), b, q, H, v_max=5.0)
        b.table[:3, :6] = b.num_pages + 3
        check_attention(run_shared(b, bounds, shared, q, H), b, q, H, v_max=5.0)


def test_shared_lowest_scores(gpu):
    """Scores of the type's lowest value and of -infinity in the prefix, ordinary ones behind it, and the other way round."""
    H, G, D = 2, 1, 64
    for dtype in (F16, F32):
        for low in (np.finfo(dtype).min, -np.inf):
            for place in (0, 1):
                b, bounds, shared = batch(6, [(64, [(1, 20), (1, 3)])], G, D, 16, dtype)
                q = np.abs(queries(b, H))
                k = b.k.reshape(-1, G, D)
                rows = [b.row(r, j) for r in range(2) for j in (range(64) if place == 0 else range(64, b.pasts[r] + 1))]
                k[rows] = low if low == -np.inf else low / dtype(64)
                log(f"low {low} {dtype.__name__} {place}")
                check_attention(run_shared(b, bounds, shared, q, H), b, q, H)


def test_groups_that_make_no_sense(gpu):
    """Bounds and lengths out of range: other groups' rows are as they should be, and nothing is read or written outside."""
    H, G, D = 4, 2, 64
    groups = [(64, [(1, 20)] * 3), (64, [(1, 5), (30, 2)]), (64, [(1, 1)] * 4)]
    b, bounds, shared = batch(7, groups, G, D, 16, F16)
    q = queries(b, H)
    want = ref.attention(b, q, H)[0]
    last = slice(int(b.cu[5]), int(b.cu[9]))
    big = 2 ** 31 - 1
    for bad, lengths in (([5, 2, 5, 9], [64, 64, 64]), ([-7, -3, 5, 9], [64, 64, 64]), ([0, 0, 5, 10 ** 6], [big, 64, 64]),
                         ([0, 3, 5, big], [-5, big, 64])):
        log(f"groups {bad} {lengths}")
        got = run_shared(b, np.array(bad, I32), np.array(lengths, I32), q, H)
        assert np.abs(got[last] - want[last]).max() < 1e-4
    cu = b.cu.copy()
    for bad in ([0, 5, 3, 9, -4, 2, 70, 7, 8, 9], [big] * 10, [-big] * 10):
        log(f"cu {bad}")
        b.cu = np.array(bad, I32)
        run_shared(b, bounds, shared, q, H)
    b.cu = cu
    b.past[:] = big
    run_shared(b, bounds, shared, q, H)
    b.past[:] = -big
    run_shared(b, bounds, shared, q, H)


def test_shared_attention_replayed_from_a_graph(gpu):
    """Captured once with roomy bounds; replays with other lengths, groups and prefixes, each as an eager call. Two
    captured graphs with workspaces of their own."""
    import torch
    H, G, D, page = 8, 2, 128, 16
    first = batch(8, [(96, [(1, 60)] * 4), (32, [(3, 9)] * 4)], G, D, page, F16, extra_columns=6)
    b, bounds, shared = first
    d = desc_of(b, H)
    s = native.SharedDesc(groups=2)
    n = native.paged_shared_attention_workspace_size(d, s)
    bufs = [dev(x) for x in (queries(b, H), b.cu, b.past, b.table, bounds, shared, b.k, b.v)]
    graphs = []
    for _ in range(2):
        out = torch.full((b.tokens, H * D), float("nan"), device="cuda")
        ws = torch.full((n // 4,), float("nan"), device="cuda")
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            native.paged_shared_attention(d, s, *map(ptr, bufs), ptr(out), ptr(ws), n, side.cuda_stream)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                native.paged_shared_attention(d, s, *map(ptr, bufs), ptr(out), ptr(ws), n, side.cuda_stream)
        graphs.append((g, out, ws))
    for i, groups in enumerate([[(96, [(1, 20)] * 4), (32, [(3, 9)] * 4)], [(16, [(1, 60)] * 2), (80, [(2, 3)] * 6)],
                                [(0, [(1, 50)] * 5), (112, [(1, 0)] * 3)]]):
        b, bounds, shared = batch(20 + i, groups, G, D, page, F16, roomy=False)
        q = np.zeros((bufs[0].shape), F32)
        q[:b.tokens] = queries(b, H)
        table = np.full(bufs[3].shape, -1, I32)
        table[:, :b.max_pages] = b.table
        cache = [np.zeros(bufs[6].shape, F16) for _ in range(2)]
        for c, x in zip(cache, (b.k, b.v)):
            c[:min(len(c), len(x))] = x[:len(c)]
        assert b.num_pages <= len(cache[0]) and b.tokens <= len(q)
        for t, x in zip(bufs, (q, b.cu, b.past, table, bounds, shared, *cache)):
            t.copy_(dev(x))
        torch.cuda.synchronize()
        for g, out, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        log(f"replay {i}")
        outs = [out.cpu().numpy()[:b.tokens] for _, out, _ in graphs]
        assert np.array_equal(outs[0], outs[1])
        check_attention(outs[0], b, q[:b.tokens], H)
