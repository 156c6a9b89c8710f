"""The serving-step operators on the GPU (paged append, paged attention, query and key norms with
rotation, low-rank adapters) against plain 64-bit forms."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import serving_ref as ref
from modelsharp_amd import native

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def log(msg):
    print(msg, flush=True)


def dev(x):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def desc_of(b, H, **kw):
    return native.PagedDesc(tokens=b.tokens, requests=len(b.news), num_heads=H, kv_num_heads=b.G, head_dim=b.D,
                            page_size=b.page, num_pages=b.num_pages, max_pages=b.max_pages,
                            cache_type=native.MS_HIP_DTYPE_F16 if b.k.dtype == F16 else native.MS_HIP_DTYPE_F32,
                            **{"local_window_size": -1, **kw})


def run_attention(b, q, H, window=-1, scale=0.0, workspace=True, hints=True, stride=0, out=None):
    """paged_attention's output; rows of no request keep `out` (else NaN)."""
    import torch
    d = desc_of(b, H, local_window_size=window, scale=scale, q_stride=stride)
    if hints:
        d.max_new, d.max_total = max(b.news), max(n + p for n, p in zip(b.news, b.pasts))
    o = torch.full((b.tokens, H * b.D), float("nan"), device="cuda") if out is None else dev(out)
    n = native.paged_attention_workspace_size(d) if workspace else 0
    ws = torch.full((n // 4 + 64,), float("nan"), device="cuda")
    bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
    native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws) if n else None, n, stream())
    torch.cuda.synchronize()
    assert torch.isnan(ws[n // 4:]).all()   # nothing past the workspace
    return o.cpu().numpy()


def finite_max(x):
    x = np.abs(x.astype(F32))
    return float(x[np.isfinite(x)].max())


def check_attention(got, b, q, H, window=-1, scale=0.0, out=None, v_max=None):
    want, mass, longest = ref.attention(b, q, H, window, scale, out)
    tol = ref.attention_tolerance(mass, longest, b.D, finite_max(b.v) if v_max is None else v_max)
    rows = np.array([t for t, _, _ in b.each_token()], int)
    assert np.array_equal(np.isnan(got[rows]), np.isnan(want[rows]))
    inf = np.isinf(want[rows])
    assert np.array_equal(got[rows][inf], want[rows][inf].astype(F32))
    fin = np.isfinite(want[rows])
    err = np.abs(got[rows][fin] - want[rows][fin]).max() if fin.any() else 0.0
    log(f"  max err {err:.2e}, tolerance {tol:.2e}")
    assert err <= tol
    rest = np.setdiff1d(np.arange(b.tokens), rows)
    if out is None:
        assert np.isnan(got[rest]).all()   # rows of no request are left as they were
    else:
        assert np.array_equal(got[rest], out[rest].astype(F32))


# news, pasts, H, G, D, page, window
ATTENTION = [
    ([1], [0], 1, 1, 8, 1, -1),                        # the smallest call: one key, a page of one row
    ([1], [700], 14, 2, 64, 16, -1),
    ([1, 1, 1, 1], [0, 15, 16, 130], 28, 4, 128, 16, -1),
    ([1] * 70, list(range(0, 210, 3)), 4, 2, 64, 8, -1),    # more requests than lanes
    ([0, 1, 0, 3, 0], [5, 9, 0, 40, 7], 8, 8, 128, 10, -1),   # requests without new tokens, odd pages
    ([5], [1000], 16, 1, 128, 64, -1),                 # 16 heads of one kv head
    ([2, 3], [50, 60], 20, 1, 40, 24, -1),             # 20 rows a token: a token's heads over two tiles
    ([33, 17], [100, 0], 6, 2, 96, 16, -1),
    ([130], [70], 12, 4, 128, 16, -1),
    ([64, 1, 100], [0, 300, 31], 28, 4, 128, 32, -1),
    ([257], [513], 7, 1, 128, 128, -1),
    ([90, 40], [45, 0], 4, 4, 256, 16, -1),
    ([75], [20], 8, 2, 80, 7, -1),
    ([200, 3, 1], [10, 333, 600], 8, 2, 64, 16, -1),
    ([1, 70], [500, 300], 8, 2, 128, 16, 100),         # sliding windows
    ([40], [90], 4, 2, 64, 10, 1),
    ([3, 20], [30, 5], 4, 2, 96, 16, 0),               # a window that shows nothing: zeros
    ([300], [0], 2, 2, 192, 16, 33),
    ([1, 2], [4500, 3000], 32, 8, 128, 256, -1),
]


@pytest.mark.parametrize("workspace", [True, False], ids=["split", "whole"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_paged_attention(gpu, case, dtype, workspace):
    news, pasts, H, G, D, page, window = ATTENTION[case]
    log(f"attention {ATTENTION[case]} {dtype.__name__} workspace={workspace}")
    b = ref.Batch(1000 + case, news, pasts, G, D, page, dtype, spare_rows=3 * (case % 2), extra_columns=case % 3)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32) * F32(1.5)
    check_attention(run_attention(b, q, H, window, workspace=workspace, hints=bool(case % 4)), b, q, H, window)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_attention_reads_packed_rows_and_takes_a_scale(gpu, dtype):
    H, G, D = 6, 2, 64
    b = ref.Batch(3, [4, 60], [33, 2], G, D, 16, dtype)
    packed = b.rng.standard_normal((b.tokens, (H + 2 * G) * D)).astype(F32)
    q = np.ascontiguousarray(packed[:, :H * D])
    check_attention(run_attention(b, packed, H, scale=0.31, stride=(H + 2 * G) * D), b, q, H, scale=0.31)


@pytest.mark.parametrize("news", [[1, 1], [40, 70]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_attention_ignores_what_it_does_not_see(gpu, dtype, news):
    """NaN and infinities in pages of nobody, behind a request's last row, in rows that later tokens
    write, and in rows before a window: the rows that do not see them are as without them."""
    H, G, D, window = 4, 2, 128, 60
    b = ref.Batch(5, news, [150, 90], G, D, 16, dtype, spare_pages=4)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    used = {b.row(r, j) for r in range(2) for j in range(b.pasts[r] + b.news[r])}
    free = np.setdiff1d(np.arange(b.num_pages * b.page), np.array(sorted(used)))
    k, v = b.k.reshape(-1, G, D), b.v.reshape(-1, G, D)
    k[free[::2]], v[free[::2]] = np.nan, np.nan
    k[free[1::2]], v[free[1::2]] = np.inf, -np.inf
    far = b.row(0, 3)                    # before every query's window
    k[far], v[far] = np.inf, np.nan
    log(f"unseen {dtype.__name__} {news}")
    got = run_attention(b, q, H, window)
    assert np.isfinite(got).all()
    check_attention(got, b, q, H, window, v_max=5.0)
    last = b.row(1, b.pasts[1] + b.news[1] - 1)   # the last token's own row: earlier tokens do not see it
    v[last] = np.nan
    got = run_attention(b, q, H, window)
    assert np.isnan(got[-1]).all() and np.isfinite(got[:-1]).all()
    check_attention(got, b, q, H, window, v_max=5.0)


@pytest.mark.parametrize("where,value", [("k", np.inf), ("k", -np.inf), ("k", np.nan), ("q", np.inf), ("q", np.nan),
                                         ("v", np.inf), ("v", -np.inf), ("v", np.nan), ("k", 6e4), ("v", 6e4)])
@pytest.mark.parametrize("news", [[1], [50]], ids=["token", "chunk"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_attention_odd_values(gpu, dtype, news, where, value):
    """One odd value: rows that see it answer as the definition does, the others are untouched."""
    H, G, D = 4, 2, 64
    b = ref.Batch(7, news, [200], G, D, 16, dtype)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    rw = b.row(0, 200 + news[0] // 2)
    if where == "q":
        q[news[0] // 2, 5] = value
    else:
        (b.k if where == "k" else b.v).reshape(-1, G, D)[rw, 1, 3] = value
    log(f"odd {where}={value} {dtype.__name__} {news}")
    check_attention(run_attention(b, q, H), b, q, H)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e20])
@pytest.mark.parametrize("news", [[2], [66]], ids=["tokens", "chunk"])
def test_attention_magnitudes(gpu, size, news):
    """fp32 caches and queries far from 1 (scores kept near 1 by the scale)."""
    H, G, D = 4, 2, 128
    b = ref.Batch(8, news, [77], G, D, 16, F32)
    b.k *= F32(size)
    b.v *= F32(size)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    log(f"magnitude {size} {news}")
    check_attention(run_attention(b, q, H, scale=float(0.1 / size) if size < 1e18 else 0.1 / size), b, q, H,
                    scale=0.1 / size)


@pytest.mark.parametrize("size", [1e-38, 1e-20, 1e30])
def test_attention_query_magnitudes_f16(gpu, size):
    H, G, D = 4, 2, 128
    for news in ([2], [66]):
        b = ref.Batch(9, news, [77], G, D, 16, F16)
        q = (b.rng.standard_normal((b.tokens, H * D)) * size).astype(F32)
        scale = float(F32(0.1 / size)) if size > 1e-37 else 1e37
        log(f"query magnitude {size} {news}")
        # below the smallest normal fp32 a query keeps fewer bits, here and in the reference's inputs
        check_attention(run_attention(b, q, H, scale=scale), b, q, H, scale=scale)


def test_attention_pages_that_are_not_there(gpu):
    for dtype in (F16, F32):
        for news in ([1, 1, 1], [50, 40, 2]):
            H, G, D = 8, 2, 128
            b = ref.Batch(11, news, [100, 37, 90], G, D, 16, dtype)
            b.table[0, 2] = -1
            b.table[0, 4] = b.num_pages
            b.table[1, :] = -5                      # nothing of this request is there: zeros
            b.table[2, 0] = 2 ** 31 - 1
            q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
            log(f"missing pages {dtype.__name__} {news}")
            got = run_attention(b, q, H)
            assert (got[b.cu[1]:b.cu[2]] == 0).all()
            check_attention(got, b, q, H)
            b.max_pages = 3                         # a table that ends before the requests do
            b.table = np.ascontiguousarray(b.table[:, :3])
            check_attention(run_attention(b, q, H), b, q, H)


def test_attention_rows_outside_every_request(gpu):
    """cu that starts behind row 0 and ends before the last: the other rows stay."""
    H, G, D = 4, 2, 64
    for news in ([1, 1], [30, 20]):
        b = ref.Batch(12, news, [600, 500], G, D, 16, F16, spare_rows=9)
        b.cu = b.cu + 4
        q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
        q[:4], q[b.cu[-1]:] = np.nan, np.nan
        out = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
        check_attention(run_attention(b, q, H, out=out), b, q, H, out=out)


@pytest.mark.parametrize("cu,past", [([0, 9, 3], [4, 4]), ([0, -5, 40], [1, 2]), ([7, 7, 100], [-3, 2 ** 31 - 1]),
                                     ([2 ** 31 - 1, 0, 5], [0, -2 ** 31])])
def test_lengths_that_make_no_sense_stay_inside(gpu, cu, past):
    """Outputs are not said, but nothing outside the buffers is read or written and the call ends."""
    import torch
    H, G, D = 4, 2, 64
    for dtype in (F16, F32):
        b = ref.Batch(13, [10, 20], [50, 60], G, D, 16, dtype)
        b.cu, b.past = np.array(cu, np.int32), np.array(past, np.int32)
        q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
        log(f"lengths {cu} {past} {dtype.__name__}")
        d = desc_of(b, H)
        n = native.paged_attention_workspace_size(d)
        ws = torch.zeros(n // 4 + 64, device="cuda")
        o = torch.zeros(b.tokens + 16, H * D, device="cuda")
        bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
        native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws), n, stream())
        torch.cuda.synchronize()
        assert (o[b.tokens:] == 0).all() and (ws[n // 4:] == 0).all()
        kv = dev(b.rng.standard_normal((b.tokens, G * D)).astype(F32))
        qo = torch.zeros(b.tokens + 16, H * D, device="cuda")
        native.paged_append(d, ptr(bufs[0]), ptr(kv), ptr(kv), None, None, *map(ptr, bufs[1:4]), None, None, ptr(qo),
                            ptr(bufs[4]), ptr(bufs[5]), stream())
        torch.cuda.synchronize()
        assert (qo[b.tokens:] == 0).all()


# ---- append and rotation -----------------------------------------------------------------------------

# news, pasts, H, G, D, page, cos_cols (0: no rotation), interleaved, norm, packed, cos_rows
APPEND = [
    ([1], [0], 1, 1, 8, 1, 4, False, True, False, 4),
    ([1, 1, 1], [0, 15, 16], 28, 4, 128, 16, 64, False, True, True, 64),
    ([1] * 70, list(range(70)), 4, 2, 64, 8, 32, True, True, False, 80),
    ([0, 5, 0, 30], [3, 10, 0, 7], 14, 2, 64, 10, 32, False, True, True, 40),
    ([20, 9], [100, 0], 8, 8, 96, 24, 24, False, True, False, 200),      # half of the channels turn
    ([20, 9], [100, 0], 8, 2, 80, 24, 40, True, False, True, 200),
    ([7], [5], 6, 3, 256, 16, 128, False, True, False, 64),
    ([7], [5], 6, 3, 256, 16, 0, False, True, False, 64),                # norms alone
    ([7], [90], 6, 3, 128, 16, 64, False, False, False, 64),             # positions past the last row
    ([11, 2], [3, 4], 3, 1, 100, 16, 50, False, True, False, 64),        # head sizes of the general kernel
    ([11, 2], [3, 4], 3, 3, 37, 5, 18, True, True, False, 64),
    ([3], [1], 2, 1, 1000, 4, 21, False, True, False, 64),
    ([3], [1], 2, 1, 64, 4, 100, False, True, False, 64),                # more columns than channels
    ([300], [40], 28, 4, 128, 16, 64, False, True, True, 512),
]


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_paged_append(gpu, case, dtype):
    import torch
    news, pasts, H, G, D, page, cols, inter, norm, packed, rows = APPEND[case]
    log(f"append {APPEND[case]} {dtype.__name__}")
    b = ref.Batch(2000 + case, news, pasts, G, D, page, dtype, spare_rows=2)
    qkv = (b.rng.standard_normal((b.tokens, (H + 2 * G) * D)) * 2).astype(F32)
    q, k, v = (np.ascontiguousarray(x) for x in np.split(qkv, [H * D, (H + G) * D], axis=1))
    gq, gk = ((b.rng.random(D) + 0.5).astype(F32) if norm else None for _ in range(2))
    ang = np.outer(np.arange(rows), 1.0 / 10000 ** (np.arange(cols) / max(cols, 1)))
    cos, sin = (np.cos(ang).astype(F32), np.sin(ang).astype(F32)) if cols else (None, None)
    d = desc_of(b, H, do_rotary=int(cols > 0), rotary_interleaved=int(inter), cos_rows=rows if cols else 0, cos_cols=cols,
                eps=1e-5)
    o = torch.full((b.tokens, H * D), float("nan"), device="cuda")
    kc, vc = dev(b.k), dev(b.v)
    keep = [dev(x) for x in (gq, gk, b.cu, b.past, b.table, cos, sin)]
    if packed:
        d.q_stride = d.k_stride = d.v_stride = (H + 2 * G) * D
        src = dev(qkv)
        rows_in = [ptr(src), ptr(src) + 4 * H * D, ptr(src) + 4 * (H + G) * D]
    else:
        src = [dev(x) for x in (q, k, v)]
        rows_in = list(map(ptr, src))
    native.paged_append(d, *rows_in, *map(ptr, keep), ptr(o), ptr(kc), ptr(vc), stream())
    torch.cuda.synchronize()
    got, wk, wv = o.cpu().numpy(), b.k.astype(np.float64), b.v.copy()
    gk_c, gv_c = kc.cpu().numpy(), vc.cpu().numpy()
    half = ref.EPS24 * (2 ** 13 if dtype == F16 else 1)   # half a step of the cache's type
    tol_q = ref.norm_tolerance(D, gq, 1.5 * np.sqrt(D) if norm else 12.0, cols > 0)
    worst, written = 0.0, np.zeros(b.num_pages * page, bool)
    for t, r, pos in b.each_token():
        want = ref.normed_rotated(q[t].reshape(H, D), gq, pos, cos, sin, inter, 1e-5)
        worst = max(worst, np.abs(got[t].reshape(H, D) - want).max())
        rw = b.row(r, pos)
        written[rw] = True
        wk.reshape(-1, G, D)[rw] = ref.normed_rotated(k[t].reshape(G, D), gk, pos, cos, sin, inter, 1e-5)
        wv.reshape(-1, G, D)[rw] = v[t].reshape(G, D).astype(dtype)
    log(f"  q err {worst:.2e}, tolerance {tol_q:.2e}")
    assert worst <= tol_q
    assert np.array_equal(gv_c, wv)                       # values are rounded once, other rows as before
    assert np.array_equal(gk_c.reshape(-1, G, D)[~written], b.k.reshape(-1, G, D)[~written])
    assert (np.abs(gk_c - wk) <= tol_q + np.abs(wk) * half * 1.01 + 2.0 ** -25 * (dtype == F16)).all()
    assert np.isnan(got[b.cu[-1]:]).all()


def test_append_drops_what_has_no_page_and_works_in_place(gpu):
    import torch
    H, G, D = 4, 2, 64
    b = ref.Batch(21, [3, 2], [14, 40], G, D, 16, F16)
    b.table[0, 1] = -1                  # positions 16 and on have no page
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    k, v = (b.rng.standard_normal((b.tokens, G * D)).astype(F32) for _ in range(2))
    gq = np.ones(D, F32)
    d = desc_of(b, H, eps=1e-6)
    qd, kc, vc = dev(q), dev(b.k), dev(b.v)
    keep = [dev(x) for x in (k, v, gq, b.cu, b.past, b.table)]
    native.paged_append(d, ptr(qd), ptr(keep[0]), ptr(keep[1]), ptr(keep[2]), None, *map(ptr, keep[3:]), None, None,
                        ptr(qd), ptr(kc), ptr(vc), stream())
    torch.cuda.synchronize()
    want_k, want_v = b.k.copy(), b.v.copy()
    for t, r, pos in b.each_token():
        rw = b.row(r, pos)
        if rw >= 0:
            want_k.reshape(-1, G, D)[rw] = k[t].reshape(G, D)
            want_v.reshape(-1, G, D)[rw] = v[t].reshape(G, D)
    assert np.array_equal(kc.cpu().numpy(), want_k) and np.array_equal(vc.cpu().numpy(), want_v)
    for t, _, pos in b.each_token():
        want = ref.normed_rotated(q[t].reshape(H, D), gq, pos, None, None, False, 1e-6)
        assert np.abs(qd.cpu().numpy()[t].reshape(H, D) - want).max() <= ref.norm_tolerance(D, gq, np.sqrt(D), False)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,H,G,D,cols,inter", [(1, 2, 1, 64, 32, False), (37, 14, 2, 64, 32, True),
                                                (260, 28, 4, 128, 64, False), (9, 3, 3, 50, 25, False),
                                                (5, 4, 2, 512, 256, False)])
def test_qk_norm_rotary(gpu, T, H, G, D, cols, inter, in_place):
    import torch
    rng = np.random.default_rng(31)
    q, k = (rng.standard_normal((T, n * D)).astype(F32) for n in (H, G))
    gq, gk = ((rng.random(D) + 0.5).astype(F32) for _ in range(2))
    pos = rng.integers(-3, 90, T).astype(np.int32)
    ang = np.outer(np.arange(80), 1.0 / 10000 ** (np.arange(cols) / cols))
    cos, sin = np.cos(ang).astype(F32), np.sin(ang).astype(F32)
    d = native.QkNormDesc(tokens=T, num_heads=H, kv_num_heads=G, head_dim=D, do_rotary=1, rotary_interleaved=int(inter),
                          cos_rows=80, cos_cols=cols, eps=1e-6)
    log(f"qk_norm_rotary {T} {H} {G} {D}")
    qd, kd = dev(q), dev(k)
    qo, ko = (qd, kd) if in_place else (torch.empty_like(qd), torch.empty_like(kd))
    keep = [dev(x) for x in (gq, gk, pos, cos, sin)]
    native.qk_norm_rotary(d, ptr(qd), ptr(kd), *map(ptr, keep), ptr(qo), ptr(ko), stream())
    torch.cuda.synchronize()
    tol = ref.norm_tolerance(D, gq, 1.5 * np.sqrt(D), True)
    for got, x, g, n in ((qo, q, gq, H), (ko, k, gk, G)):
        want = np.stack([ref.normed_rotated(x[t].reshape(n, D), g, int(pos[t]), cos, sin, inter, 1e-6) for t in range(T)])
        assert np.abs(got.cpu().numpy().reshape(T, n, D) - want).max() <= tol


@pytest.mark.parametrize("D", [64, 50])
@pytest.mark.parametrize("norm", [False, True])
def test_qk_norm_without_rotation_reads_no_positions_and_no_caches(gpu, D, norm):
    """do_rotary = 0: positions, cos and sin may be null, and so may either norm's weights."""
    import torch
    T, H, G = 5, 4, 2
    rng = np.random.default_rng(33)
    q, k = (rng.standard_normal((T, n * D)).astype(F32) for n in (H, G))
    gk = (rng.random(D) + 0.5).astype(F32) if norm else None
    d = native.QkNormDesc(tokens=T, num_heads=H, kv_num_heads=G, head_dim=D, eps=1e-6)
    log(f"qk_norm without rotation D={D} norm={norm}")
    qd, kd, gd = dev(q), dev(k), dev(gk)
    qo, ko = torch.empty_like(qd), torch.empty_like(kd)
    native.qk_norm_rotary(d, ptr(qd), ptr(kd), None, ptr(gd), None, None, None, ptr(qo), ptr(ko), stream())
    torch.cuda.synchronize()
    assert np.array_equal(qo.cpu().numpy(), q)
    want = np.stack([ref.normed_rotated(k[t].reshape(G, D), gk, 0, None, None, False, 1e-6) for t in range(T)])
    tol = ref.norm_tolerance(D, gk, 1.5 * np.sqrt(D), False)
    assert np.abs(ko.cpu().numpy().reshape(T, G, D) - want).max() <= tol


# ---- low-rank adapters -----------------------------------------------------------------------------

# T, K, N, adapters, max_rank, pattern of adapters, with ranks / scales, base ("new", "same", None)
LORA = [
    (1, 64, 64, 1, 1, "all", False, "new"),
    (1, 4096, 1000, 3, 16, "all", True, "new"),
    (7, 100, 52, 3, 5, "mixed", True, "new"),            # nothing divides
    (16, 256, 256, 16, 8, "each", True, "same"),          # every token its own adapter
    (33, 896, 300, 5, 20, "mixed", True, "new"),
    (64, 512, 128, 40, 16, "each", True, None),
    (65, 264, 264, 4, 64, "runs", True, "same"),
    (300, 1024, 520, 4, 64, "runs", True, "new"),
    (130, 96, 2000, 2, 130, "mixed", True, "new"),        # several groups of rank tiles
    (200, 3000, 72, 7, 32, "mixed", False, None),
    (20, 128, 64, 2, 8, "none", True, "new"),             # no token has an adapter
    (20, 128, 64, 2, 8, "none", True, None),
    (1100, 96, 300, 5, 20, "mixed", True, "new"),         # many tiles
    (1040, 1024, 264, 4, 64, "runs", True, "same"),
    (1033, 100, 52, 3, 5, "mixed", True, "new"),
    (1030, 64, 520, 3, 130, "mixed", True, None),
    (2100, 160, 2056, 6, 16, "runs", True, "new"),
    (1029, 64, 64, 2, 8, "none", True, "same"),
]


def lora_inputs(case, dtype, seed):
    T, K, N, A, R, pattern, extra, base = case
    rng = np.random.default_rng(seed)
    a = (rng.standard_normal((A, R, K)) / np.sqrt(K)).astype(dtype)
    b = (rng.standard_normal((A, N, R)) * 0.3).astype(dtype)
    which = {"all": np.zeros(T, int), "each": np.arange(T) % A, "none": np.full(T, -1),
             "mixed": rng.integers(-1, A + 1, T), "runs": np.arange(T) * A // T}[pattern].astype(np.int32)
    ranks = rng.integers(0, R + 1, A).astype(np.int32) if extra else None
    if ranks is not None:
        ranks[0] = R
        for i in range(A):   # nothing past an adapter's rank is read as a value
            a[i, ranks[i]:], b[i, :, ranks[i]:] = np.nan, np.inf
    scales = (rng.random(A) + 0.5).astype(F32) if extra else None
    x = rng.standard_normal((T, K)).astype(F32)
    y0 = rng.standard_normal((T, N)).astype(F32) if base else None
    return x, a, b, ranks, scales, which, y0


def run_lora(case, x, a, b, ranks, scales, which, y0, same):
    import torch
    T, K, N, A, R = case[:5]
    d = native.LoraDesc(tokens=T, K=K, N=N, adapters=A, max_rank=R,
                        weight_type=native.MS_HIP_DTYPE_F16 if a.dtype == F16 else native.MS_HIP_DTYPE_F32)
    n = native.lora_workspace_size(d)
    ws = torch.full((n // 4 + 64,), float("nan"), device="cuda")
    base = dev(y0)
    y = base if same else torch.full((T, N), float("nan"), device="cuda")
    keep = [dev(v) for v in (x, a, b, ranks, scales, which)]
    native.lora(d, *map(ptr, keep), ptr(base), ptr(y), ptr(ws), n, stream())
    torch.cuda.synchronize()
    assert torch.isnan(ws[n // 4:]).all()
    return y.cpu().numpy()


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", LORA, ids=lambda c: "-".join(map(str, c)))
def test_lora(gpu, case, dtype):
    log(f"lora {case} {dtype.__name__}")
    x, a, b, ranks, scales, which, y0 = lora_inputs(case, dtype, 41)
    want, terms = ref.lora(x, a, b, ranks, scales, which, y0)
    got = run_lora(case, x, a, b, ranks, scales, which, y0, case[7] == "same")
    tol = ref.lora_tolerance(want, terms, case[1], case[4])
    log(f"  worst err / tolerance {np.max(np.abs(got - want) / tol):.3f}")
    assert (np.abs(got - want) <= tol).all()
    none = (which < 0) | (which >= case[3])
    assert np.array_equal(got[none], np.zeros_like(got[none]) if y0 is None else y0[none])


def test_lora_keeps_a_tokens_odd_values_to_itself(gpu):
    case = (40, 256, 128, 3, 16, "mixed", True, "new")
    x, a, b, ranks, scales, which, y0 = lora_inputs(case, F16, 43)
    which[:] = np.arange(40) % 3
    clean = run_lora(case, x, a, b, ranks, scales, which, y0, False)
    x[5, 7], x[20, 3], x[6, 1] = np.nan, np.inf, np.nan   # token 6's adapter has its whole rank
    got = run_lora(case, x, a, b, ranks, scales, which, y0, False)
    with np.errstate(invalid="ignore"):
        want, _ = ref.lora(x, a, b, ranks, scales, which, y0)
    rest = np.setdiff1d(np.arange(40), [5, 6, 20])
    assert np.array_equal(got[rest], clean[rest])
    assert np.isnan(got[6]).all() and np.array_equal(np.isnan(got[5]), np.isnan(want[5]))   # rank 0: the base


# ---- graph nodes and a run of them together -------------------------------------------------------------

def host(t):
    return t.cpu().numpy() if hasattr(t, "cpu") else t


def rotary_caches(rows, half):
    ang = np.outer(np.arange(rows), 1.0 / 10000 ** (np.arange(half) / half))
    return np.cos(ang).astype(F32), np.sin(ang).astype(F32)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_attention_block_of_a_serving_step(gpu, dtype):
    """LoraMatMulNBits (q, k, v) -> PagedAttention with norms and rotation -> LoraMatMulNBits (o), as a graph
    run by the engine: two prompts in two chunks each, then single tokens, a third request joining
    late. Every node is checked in 64 bits on what it was given."""
    import torch
    from modelsharp_amd import pipeline, workloads
    from modelsharp_amd.graph import GraphNode, ModelGraph
    E, H, G, D, page, R, pages, rows = 256, 8, 2, 64, 16, 3, 24, 96
    rng = np.random.default_rng(77)
    init, dequant = {}, {}
    nodes = []
    for name, K, N, x, y in (("qkv", E, (H + 2 * G) * D, "x", "p"), ("o", H * D, E, "attn", "y")):
        w, s, z = workloads.make_weights(workloads.Op(name, K, N, 32, True), seed=N)
        a = (rng.standard_normal((2, 8, K)) / np.sqrt(K)).astype(F16)
        b = (rng.standard_normal((2, N, 8)) * 0.1).astype(F16)
        init.update({name + ".b": w, name + ".s": s, name + ".z": z, name + ".la": a, name + ".lb": b,
                     name + ".r": np.array([8, 5], np.int32), name + ".ls": np.array([1.0, 2.0], F32)})
        nodes.append(GraphNode("LoraMatMulNBits", name, [x] + [name + e for e in (".b", ".s", ".z", ".la", ".lb", ".r",
                                                                                  ".ls")] + ["which"], [y],
                               {"K": K, "N": N, "bits": 4, "block_size": 32}))
        h = native.NBitsWeights(w, s, z, N, K, 4, 32)
        dequant[name] = h.dequant().astype(np.float64)
        h.close()
    cos, sin = rotary_caches(rows, D // 2)
    init.update({"cos": cos, "sin": sin, "gq": (rng.random(D) + 0.5).astype(F32), "gk": (rng.random(D) + 0.5).astype(F32)})
    nodes.insert(1, GraphNode("PagedAttention", "attn", ["p", "", "", "kc", "vc", "cu", "past", "table", "cos", "sin", "gq",
                                                         "gk"], ["attn", "kc2", "vc2"],
                              {"num_heads": H, "kv_num_heads": G, "do_rotary": 1, "epsilon": 1e-6}))
    engine = pipeline.build(ModelGraph(nodes, init, [], ["p", "attn", "y", "kc2"]))
    kc, vc = (torch.zeros(pages, page, G, D, dtype=torch.float16 if dtype == F16 else torch.float32, device="cuda")
              for _ in range(2))
    past = np.zeros(R, int)
    table = rng.permutation(pages).reshape(R, pages // R).astype(np.int32)
    for step, news in enumerate(([9, 5, 0], [2, 14, 0], [1, 1, 7], [1, 0, 1], [1, 1, 1])):
        T = sum(news)
        log(f"step {step}: new {news}, past {past.tolist()}")
        which = np.repeat([0, -1, 1], news).astype(np.int32)
        x = rng.standard_normal((T, E)).astype(F32)
        feeds = {"x": dev(x), "kc": kc, "vc": vc, "cu": np.concatenate([[0], np.cumsum(news)]).astype(np.int32),
                 "past": past.astype(np.int32), "table": table, "which": which}
        if step % 2:   # lengths on the device as well as on the host
            feeds.update({k: dev(feeds[k]) for k in ("cu", "past", "table", "which")})
        before_k, before_v = host(kc).copy(), host(vc).copy()
        out = engine.run(feeds)
        p, attn, y = (host(out[k]) for k in ("p", "attn", "y"))
        assert out["kc2"].data_ptr() == kc.data_ptr()
        for name, src, got in (("qkv", x, p), ("o", attn, y)):
            want, terms = ref.lora(src, init[name + ".la"], init[name + ".lb"], init[name + ".r"], init[name + ".ls"],
                                   which, src.astype(np.float64) @ dequant[name].T)
            scale = np.abs(src.astype(np.float64)) @ np.abs(dequant[name]).T + terms
            # fp32-level products (up to 16 tokens): K roundings of the sum of magnitudes at the most
            assert (np.abs(got - want) <= scale * (src.shape[1] / 8 + 32) * ref.EPS24).all()
        b = ref.Batch(0, news, past, G, D, page, dtype)
        b.num_pages, b.max_pages, b.table, b.k, b.v = pages, table.shape[1], table, host(kc), host(vc)
        q = np.zeros((T, H * D), F32)
        half = ref.EPS24 * (2 ** 13 if dtype == F16 else 1)
        for t, r, pos in b.each_token():
            q[t] = ref.normed_rotated(p[t, :H * D].reshape(H, D), init["gq"], pos, cos, sin, False, 1e-6).reshape(-1)
            k = ref.normed_rotated(p[t, H * D:(H + G) * D].reshape(G, D), init["gk"], pos, cos, sin, False, 1e-6)
            tol = ref.norm_tolerance(D, init["gk"], 1.5 * np.sqrt(D), True)
            rw = b.row(r, pos)
            assert (np.abs(b.k.reshape(-1, G, D)[rw] - k) <= tol + np.abs(k) * half * 1.01 + 2.0 ** -25).all()
            assert np.array_equal(b.v.reshape(-1, G, D)[rw], p[t, (H + G) * D:].reshape(G, D).astype(dtype))
            before_k.reshape(-1, G, D)[rw], before_v.reshape(-1, G, D)[rw] = b.k.reshape(-1, G, D)[rw], \
                b.v.reshape(-1, G, D)[rw]
        assert np.array_equal(b.k, before_k) and np.array_equal(b.v, before_v)   # nothing else was written
        want, mass, longest = ref.attention(b, q, H)
        # the queries themselves are off by their norm's tolerance, relative to their largest value
        tol = ref.attention_tolerance(mass, longest, D, float(np.abs(b.v).max()))
        tol += 2 * mass * ref.norm_tolerance(D, init["gq"], 1.0, True) * float(np.abs(b.v).max()) * np.sqrt(D)
        assert np.abs(attn - want).max() <= tol
        past = past + news


def test_nodes_for_group_query_attention(gpu):
    """QkNormRotary before GroupQueryAttention without rotation gives what the norm on the host before
    GroupQueryAttention with rotation gives."""
    from modelsharp_amd.decoder_kernels import HipGroupQueryAttentionKernel
    from modelsharp_amd.graph import GraphContext, GraphNode
    from modelsharp_amd.serving_kernels import HipQkNormRotaryKernel
    rng = np.random.default_rng(5)
    S, H, G, D = 20, 4, 2, 64
    q, k, v = (rng.standard_normal((1, S, n * D)).astype(F32) for n in (H, G, G))
    gq, gk = ((rng.random(D) + 0.5).astype(F32) for _ in range(2))
    cos, sin = rotary_caches(32, D // 2)
    ctx = GraphContext({"q": q, "k": k, "v": v, "gq": gq, "gk": gk, "pos": np.arange(S)[None], "cos": cos, "sin": sin})
    HipQkNormRotaryKernel().execute(GraphNode("QkNormRotary", "r", ["q", "k", "gq", "gk", "pos", "cos", "sin"],
                                              ["q2", "k2"], {"num_heads": H, "kv_num_heads": G}), ctx)
    attrs = {"num_heads": H, "kv_num_heads": G}
    HipGroupQueryAttentionKernel().execute(GraphNode("GroupQueryAttention", "a", ["q2", "k2", "v"], ["o"], attrs), ctx)
    normed = GraphContext({"v": v, "cos": cos, "sin": sin,
                           **{n: ref.normed_rotated(x.reshape(-1, D), g, 0, None, None, False, 1e-6).reshape(x.shape)
                              .astype(F32) for n, x, g in (("q", q, gq), ("k", k, gk))}})
    HipGroupQueryAttentionKernel().execute(GraphNode("GroupQueryAttention", "b", ["q", "k", "v", "", "", "", "", "cos", "sin"],
                                                     ["o"], {**attrs, "do_rotary": 1}), normed)
    got, want = host(ctx.get_tensor("o")), host(normed.get_tensor("o"))
    # two fp32 chains of the same definition: each within the attention's tolerance of 64 bits
    assert np.abs(got - want).max() <= 2 * ref.attention_tolerance(2 * D, S, D, np.abs(v).max())


# ---- captured, on other streams, twice --------------------------------------------------------------------

class _Step:
    """A step's buffers: append, attention and an adapter on what they leave."""

    def __init__(self, seed, news, pasts, dtype=F16, H=8, G=2, D=128):
        import torch
        self.b = b = ref.Batch(seed, news, pasts, G, D, 16, dtype, extra_columns=4, spare_pages=8)
        b.table[b.table < 0] = 0
        rng = b.rng
        self.H, T = H, b.tokens
        self.d = desc_of(b, H, eps=1e-6)
        self.d.q_stride = self.d.k_stride = self.d.v_stride = (H + 2 * G) * D
        self.da = desc_of(b, H)
        self.qkv = dev(rng.standard_normal((T, (H + 2 * G) * D)).astype(F32))
        self.cu, self.past, self.table, self.k, self.v = (dev(x) for x in (b.cu, b.past, b.table, b.k, b.v))
        self.gq = dev((rng.random(D) + 0.5).astype(F32))
        self.q, self.out = (torch.zeros(T, H * D, device="cuda") for _ in range(2))
        self.dl = native.LoraDesc(tokens=T, K=H * D, N=256, adapters=3, max_rank=16, weight_type=native.MS_HIP_DTYPE_F16)
        self.la, self.lb = dev(rng.standard_normal((3, 16, H * D)).astype(F16)), dev(rng.standard_normal((3, 256, 16)).astype(F16))
        self.which = dev((np.arange(T) % 4 - 1).astype(np.int32))
        self.y = torch.zeros(T, 256, device="cuda")
        self.n, self.nl = native.paged_attention_workspace_size(self.da), native.lora_workspace_size(self.dl)
        self.ws, self.wl = (torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in (self.n, self.nl))

    def run(self):
        st, q = stream(), ptr(self.qkv)
        k = q + 4 * self.H * self.b.D
        native.paged_append(self.d, q, k, k + 4 * self.b.G * self.b.D, ptr(self.gq), ptr(self.gq), ptr(self.cu),
                            ptr(self.past), ptr(self.table), None, None, ptr(self.q), ptr(self.k), ptr(self.v), st)
        native.paged_attention(self.da, ptr(self.q), ptr(self.cu), ptr(self.past), ptr(self.table), ptr(self.k), ptr(self.v),
                               ptr(self.out), ptr(self.ws), self.n, st)
        native.lora(self.dl, ptr(self.out), ptr(self.la), ptr(self.lb), None, None, ptr(self.which), None, ptr(self.y),
                    ptr(self.wl), self.nl, st)

    def results(self):
        import torch
        torch.cuda.synchronize()
        return [x.cpu().numpy().copy() for x in (self.q, self.out, self.y, self.k, self.v)]


@pytest.mark.parametrize("news,pasts", [([1] * 5, [300, 0, 77, 600, 16]), ([60, 1, 100], [40, 500, 0])],
                         ids=["tokens", "chunks"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_a_captured_step_replays_with_new_lengths_and_inputs(gpu, dtype, news, pasts):
    import torch
    s = _Step(51, news, pasts, dtype)
    s.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run()
    rng = np.random.default_rng(52)
    for replay in range(4):
        log(f"replay {replay} {dtype.__name__} {news}")
        s.qkv.copy_(dev(rng.standard_normal(s.qkv.shape).astype(F32)))
        if replay:   # the tokens go round the requests, the histories shrink
            new = np.roll(news, replay)
            s.cu.copy_(dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)))
            s.past.copy_(dev((np.asarray(pasts) // (replay + 1)).astype(np.int32)))
        k0, v0 = s.k.clone(), s.v.clone()
        for x in (s.q, s.out, s.y):
            x.fill_(float("nan"))
        g.replay()
        got = s.results()
        s.k.copy_(k0)
        s.v.copy_(v0)
        for x in (s.q, s.out, s.y):
            x.fill_(float("nan"))
        s.run()
        for a, b in zip(got, s.results()):
            assert np.array_equal(a, b, equal_nan=True)   # the same launches: bit for bit


def test_steps_on_two_streams_at_once(gpu):
    import torch
    steps = [_Step(61, [1] * 4, [900, 500, 40, 0]), _Step(62, [70, 30], [100, 0])]
    want = []
    for s in steps:
        k0, v0 = s.k.clone(), s.v.clone()
        s.run()
        want.append(s.results())
        s.k.copy_(k0)
        s.v.copy_(v0)
        for x in (s.q, s.out, s.y):
            x.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(10):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.run()
    for s, w in zip(steps, want):
        for a, b in zip(s.results(), w):
            assert np.array_equal(a, b)


def test_results_do_not_depend_on_the_hints_within_tolerance_and_repeat_exactly(gpu):
    H, G, D = 8, 2, 128
    for news, pasts in (([1, 1], [1000, 30]), ([90, 2], [100, 800])):
        b = ref.Batch(71, news, pasts, G, D, 16, F16)
        q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
        for hints in (True, False):
            one = run_attention(b, q, H, hints=hints)
            check_attention(one, b, q, H)
            assert np.array_equal(one, run_attention(b, q, H, hints=hints))
        # bounds that are wrong still leave right results
        import torch
        d = desc_of(b, H, max_new=1, max_total=5)
        n = native.paged_attention_workspace_size(d)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
        o = torch.full((b.tokens, H * D), float("nan"), device="cuda")
        native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws), n, stream())
        check_attention(host(o), b, q, H)


# ---- alignment, offsets, small numbers -----------------------------------------------------------------

def shifted(x):
    """A device copy that starts 4 bytes into its allocation."""
    import torch
    t = torch.empty(x.size + 1, dtype=torch.from_numpy(x).dtype, device="cuda")
    v = t[1:].view(x.shape)
    v.copy_(dev(x))
    return v


@pytest.mark.parametrize("news", [[1, 2], [60]], ids=["tokens", "chunk"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_rows_aligned_to_four_bytes(gpu, dtype, news):
    import torch
    H, G, D = 8, 2, 128
    pasts = [200] * len(news)
    b = ref.Batch(81, news, pasts, G, D, 16, dtype)
    q, k, v = (b.rng.standard_normal((b.tokens, n * D)).astype(F32) for n in (H, G, G))
    gq, gk = ((b.rng.random(D) + 0.5).astype(F32) for _ in range(2))
    cos, sin = rotary_caches(300, D // 2)
    d = desc_of(b, H, eps=1e-6, do_rotary=1, cos_rows=300, cos_cols=D // 2)
    outs = []
    for put in (dev, shifted):
        src = [put(x) for x in (q, k, v, gq, gk)]
        lens = [dev(x) for x in (b.cu, b.past, b.table)]
        rot = [put(x) for x in (cos, sin)]
        o, kc, vc = put(np.zeros_like(q)), dev(b.k), dev(b.v)
        native.paged_append(d, *map(ptr, src), *map(ptr, lens), *map(ptr, rot), ptr(o), ptr(kc), ptr(vc), stream())
        n = native.paged_attention_workspace_size(d)
        ws, out = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), put(np.zeros_like(q))
        native.paged_attention(d, ptr(o), *map(ptr, lens), ptr(kc), ptr(vc), ptr(out), ptr(ws), n, stream())
        outs.append([host(x) for x in (o, kc, out)])
    # two orders of the norm's sum of squares: the chunks' queries and keys differ in a few last bits
    tol = 2 * ref.norm_tolerance(D, gq, 1.5 * np.sqrt(D), True)
    assert np.abs(outs[0][0] - outs[1][0]).max() <= tol
    assert (np.abs(outs[0][1].astype(F32) - outs[1][1]) <= tol + np.abs(outs[0][1].astype(F32)) * (2.0 ** -10 if dtype == F16 else 0)).all()
    for o, kc, out in outs:
        b.k, b.v = kc, host(vc)
        check_attention(out, b, o, H)


@pytest.mark.parametrize("T", [5, 1040])
def test_lora_rows_aligned_to_their_type(gpu, T):
    import torch
    case = (T, 96, 68, 2, 20, "mixed", True, "new")
    x, a, b, ranks, scales, which, y0 = lora_inputs(case, F16, 83)
    want, terms = ref.lora(x, a, b, ranks, scales, which, y0)
    d = native.LoraDesc(tokens=T, K=96, N=68, adapters=2, max_rank=20, weight_type=native.MS_HIP_DTYPE_F16)
    n = native.lora_workspace_size(d)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    half = torch.empty(a.size + b.size + 2, dtype=torch.float16, device="cuda")
    half[1:1 + a.size], half[2 + a.size:] = dev(a).reshape(-1), dev(b).reshape(-1)
    y = shifted(np.zeros_like(y0))
    keep = [shifted(v) for v in (x, ranks, scales, which, y0)]
    native.lora(d, ptr(keep[0]), half.data_ptr() + 2, half.data_ptr() + 2 * (2 + a.size), *map(ptr, keep[1:]), ptr(y), ptr(ws),
                n, stream())
    assert (np.abs(host(y) - want) <= ref.lora_tolerance(want, terms, 96, 20)).all()


@pytest.mark.parametrize("news", [[1], [40]], ids=["token", "chunk"])
def test_pages_past_two_to_the_31_elements(gpu, news):
    """The same pages in a small cache and behind 2^31 elements of a large one: the same bits."""
    import torch
    H, G, D, page = 16, 8, 256, 64
    b = ref.Batch(85, news, [130], G, D, page, F16)
    far = 2 ** 31 // (page * G * D) + 1          # the first page behind
    q, k, v = (b.rng.standard_normal((b.tokens, n * D)).astype(F32) for n in (H, G, G))
    outs = []
    for shift in (0, far):
        kc, vc = (torch.zeros(b.num_pages + shift, page, G, D, dtype=torch.float16, device="cuda") for _ in range(2))
        kc[shift:], vc[shift:] = dev(b.k), dev(b.v)
        d = desc_of(b, H, eps=1e-6)
        d.num_pages = b.num_pages + shift
        lens = [dev(x) for x in (b.cu, b.past, np.where(b.table >= 0, b.table + shift, -1).astype(np.int32))]
        src, qo = [dev(x) for x in (q, k, v)], torch.zeros(b.tokens, H * D, device="cuda")
        native.paged_append(d, *map(ptr, src), None, None, *map(ptr, lens), None, None, ptr(qo), ptr(kc), ptr(vc), stream())
        n = native.paged_attention_workspace_size(d)
        ws, out = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), torch.zeros_like(qo)
        native.paged_attention(d, ptr(qo), *map(ptr, lens), ptr(kc), ptr(vc), ptr(out), ptr(ws), n, stream())
        outs.append([host(out), host(kc[shift:]), host(vc[shift:])])
        del kc, vc
    for x, y in zip(*outs):
        assert np.array_equal(x, y)
    b.k, b.v = outs[0][1:]
    check_attention(outs[0][0], b, q, H)


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("news", [[2], [66]], ids=["tokens", "chunk"])
def test_attention_subnormal_fp16_values(gpu, news, where):
    H, G, D = 4, 2, 128
    b = ref.Batch(87, news, [77], G, D, 16, F16)
    x = (b.rng.standard_normal(b.k.shape) * 2e-6).astype(F16)   # most below fp16's smallest normal value
    if where == "k":
        b.k = x
    else:
        b.v = x
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    scale = 5e4 if where == "k" else 0.0
    check_attention(run_attention(b, q, H, scale=scale), b, q, H, scale=scale)


def test_many_tiles_of_adapters_captured(gpu):
    import torch
    case = (1100, 256, 132, 3, 64, "runs", True, "new")
    x, a, b, ranks, scales, which, y0 = lora_inputs(case, F16, 89)
    want, terms = ref.lora(x, a, b, ranks, scales, which, y0)
    d = native.LoraDesc(tokens=1100, K=256, N=132, adapters=3, max_rank=64, weight_type=native.MS_HIP_DTYPE_F16)
    n = native.lora_workspace_size(d)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    keep = [dev(v) for v in (x, a, b, ranks, scales, which, y0)]
    y = torch.empty_like(keep[-1])
    g = torch.cuda.CUDAGraph()
    call = lambda: native.lora(d, *map(ptr, keep), ptr(y), ptr(ws), n, stream())   # noqa: E731
    call()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        call()
    for replay in range(4):
        y.fill_(float("nan"))
        ws.fill_(255)
        torch.cuda.synchronize()
        g.replay()
        got = host(y)
        assert (np.abs(got - want) <= ref.lora_tolerance(want, terms, 256, 64)).all()
        y.fill_(float("nan"))
        call()
        assert np.array_equal(host(y), got)


# Around the borders of the launch rules: rows of a request in tiles of 16 or of 128, keys kept together or
# split.
BORDERS = [
    ([9, 10, 18, 19], [300, 40, 0, 700], 28, 4, 128, 16, -1),   # 63 to 133 rows
    ([1, 9], [600, 500], 28, 4, 128, 16, -1),
    ([36], [513], 28, 4, 128, 16, -1),                  # 252 rows, few tokens: tiles of 16
    ([37], [513], 28, 4, 128, 24, -1),
    ([128], [30], 8, 1, 64, 16, -1),                    # 1024 rows of few tokens
    ([30, 2, 96], [100, 5, 0], 8, 1, 64, 10, -1),       # 240, 16 and 768 of them
    ([1], [511], 4, 4, 128, 16, -1),
    ([1], [512], 4, 4, 128, 16, -1),
    ([1, 0, 1], [0, 9000, 9000], 2, 1, 64, 64, -1),     # a request of one key beside one of many splits
    ([16, 17], [800, 20], 32, 8, 128, 32, -1),
    ([32, 33, 1], [50, 400, 3], 32, 8, 96, 16, -1),     # 128 and 132 rows
    ([48, 1], [2000, 2000], 8, 1, 96, 10, 700),
]


@pytest.mark.parametrize("hints", [True, False], ids=["bounds", "no-bounds"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(BORDERS)))
def test_paged_attention_around_the_launch_rules(gpu, case, dtype, hints):
    news, pasts, H, G, D, page, window = BORDERS[case]
    log(f"attention {BORDERS[case]} {dtype.__name__} bounds={hints}")
    b = ref.Batch(2000 + case, news, pasts, G, D, page, dtype, spare_rows=case % 2)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32) * F32(1.5)
    check_attention(run_attention(b, q, H, window, hints=hints), b, q, H, window)


def test_bounds_that_are_too_small_cost_no_result(gpu):
    """max_new and max_total choose the launch only."""
    import torch
    b = ref.Batch(91, [1, 150, 9], [700, 20, 300], 2, 64, 16, F16)
    q = b.rng.standard_normal((b.tokens, 8 * 64)).astype(F32)
    for new, total in [(1, 1), (1, 10 ** 6), (200, 8), (2 ** 31 - 1, 2 ** 31 - 1)]:
        d = desc_of(b, 8, max_new=new, max_total=total)
        n = native.paged_attention_workspace_size(d)
        ws = torch.full((n // 4 + 64,), float("nan"), device="cuda")
        o = torch.full((b.tokens, 8 * 64), float("nan"), device="cuda")
        bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
        native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws), n, stream())
        check_attention(host(o), b, q, 8)
        assert torch.isnan(ws[n // 4:]).all()


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", [
    (128, 256, 264, 20, 16, "each", True, "new"),        # the last of few tiles
    (129, 256, 264, 20, 16, "each", True, "new"),        # classes over workgroups
    (144, 520, 300, 16, 16, "each", True, "same"),
    (160, 264, 264, 5, 64, "mixed", True, "new"),
    (400, 96, 72, 30, 130, "each", True, None),
    (513, 100, 52, 20, 20, "each", True, "new"),
], ids=lambda c: "-".join(map(str, c)))
def test_lora_around_the_launch_rules(gpu, case, dtype):
    test_lora(gpu, case, dtype)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", [
    (40, 264, 132, 5, 20, "mixed", True, "new"),         # ranks of whole fours
    (40, 100, 132, 5, 20, "mixed", True, "same"),        # x in single values, y in chunks
    (40, 264, 131, 5, 20, "mixed", True, "new"),         # and the other way
    (40, 264, 132, 5, 19, "mixed", True, "new"),
    (640, 264, 132, 5, 100, "runs", True, "new"),
    (640, 100, 132, 5, 36, "mixed", True, "new"),
    (640, 264, 130, 5, 4, "mixed", True, None),
], ids=lambda c: "-".join(map(str, c)))
def test_lora_in_whole_chunks_on_either_side(gpu, case, dtype):
    test_lora(gpu, case, dtype)


def test_node_inputs_on_the_host_follow_the_first_ones_device(gpu):
    import torch
    from modelsharp_amd import workloads
    from modelsharp_amd.graph import GraphContext, GraphNode
    from modelsharp_amd.serving_kernels import HipLoraMatMulNBitsKernel, HipQkNormRotaryKernel
    rng = np.random.default_rng(6)
    w, s, z = workloads.make_weights(workloads.Op("p", 64, 96, 32, True), seed=1)
    cos, sin = rotary_caches(32, 32)
    values = {"q": rng.standard_normal((5, 256)).astype(F32), "k": rng.standard_normal((5, 128)).astype(F32),
              "g": (rng.random(64) + 0.5).astype(F32), "pos": np.arange(5, dtype=np.int32), "cos": cos, "sin": sin,
              "x": rng.standard_normal((5, 64)).astype(F32), "la": rng.standard_normal((2, 8, 64)).astype(F16),
              "lb": rng.standard_normal((2, 96, 8)).astype(F16), "r": np.array([8, 3], np.int32),
              "ls": np.array([1.0, 0.5], F32), "which": np.array([0, 1, -1, 1, 0], np.int32)}
    results = []
    for place in (dev, torch.from_numpy):
        ctx = GraphContext({"b": w, "s": s, "z": z,
                            **{n: (dev if n in "qx" else place)(v) for n, v in values.items()}})
        HipQkNormRotaryKernel().execute(GraphNode("QkNormRotary", "r", ["q", "k", "g", "g", "pos", "cos", "sin"],
                                                  ["q2", "k2"], {"num_heads": 4, "kv_num_heads": 2}), ctx)
        k = HipLoraMatMulNBitsKernel()
        k.execute(GraphNode("LoraMatMulNBits", "l", ["x", "b", "s", "z", "la", "lb", "r", "ls", "which"], ["y"],
                            {"K": 64, "N": 96, "bits": 4, "block_size": 32}), ctx)
        results.append([host(ctx.get_tensor(n)) for n in ("q2", "k2", "y")])
        k.close()
    assert all(np.array_equal(a, b) and np.isfinite(a).all() for a, b in zip(*results))
