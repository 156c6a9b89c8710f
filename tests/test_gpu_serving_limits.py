"""The serving-step operators on the GPU at the borders of what their entries take: workspaces,
lengths, pages that are not there."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from modelsharp_amd import native
from test_gpu_serving import F16, F32, check_attention, desc_of, dev, host, log, ptr, run_attention, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [-1, -2 ** 31, 0, 16])
def test_a_workspace_that_is_too_small_is_not_written(gpu, size):
    import torch
    H, G, D = 8, 2, 64
    b = ref.Batch(101, [1, 1], [3000, 40], G, D, 16, F16)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    d = desc_of(b, H)
    n = native.paged_attention_workspace_size(d)
    assert n > 16   # with a workspace the keys are shared out
    log(f"workspace of {size} bytes")
    ws = torch.full((n // 4 + 64,), float("nan"), device="cuda")
    o = torch.full((b.tokens, H * D), float("nan"), device="cuda")
    bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
    native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws), size, stream())
    check_attention(host(o), b, q, H)
    assert torch.isnan(ws).all()


@pytest.mark.parametrize("cu", [[2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -2 ** 31],
                                [2 ** 31 - 1, -2 ** 31, 30]])
def test_lengths_that_wrap_stay_inside(gpu, cu):
    """Outputs are not said, but nothing outside the buffers is read or written and the call ends."""
    import torch
    H, G, D = 4, 2, 64
    for dtype in (F16, F32):
        b = ref.Batch(103, [10, 20], [50, 60], G, D, 16, dtype)
        b.cu = np.array(cu, np.int32)
        q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
        log(f"lengths {cu} {dtype.__name__}")
        d = desc_of(b, H)
        n = native.paged_attention_workspace_size(d)
        ws = torch.zeros(n // 4 + 64, device="cuda")
        o = torch.zeros(b.tokens + 16, H * D, device="cuda")
        bufs = [dev(x) for x in (q, b.cu, b.past, b.table, b.k, b.v)]
        native.paged_attention(d, *map(ptr, bufs), ptr(o), ptr(ws), n, stream())
        torch.cuda.synchronize()
        assert (o[b.tokens:] == 0).all() and (ws[n // 4:] == 0).all()


@pytest.mark.parametrize("first", [2 ** 30 - 20, 2 ** 30 + 70000, 2 ** 31 - 4096 - 90], ids=["2^30", "past-2^30", "last"])
@pytest.mark.parametrize("news", [[2], [90]], ids=["tokens", "chunk"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_positions_of_a_very_long_history(gpu, dtype, news, first):
    """Appends and attention under a window agree about positions past 2^30, where only the last pages
    are there."""
    import torch
    H, G, D, page, window = 4, 1, 64, 1 << 16, 70
    b = ref.Batch(105, news, [1], G, D, page, dtype, spare_pages=1)
    b.pasts, b.past = [first], np.array([first], np.int32)
    b.max_pages = (first + news[0] - 1) // page + 1
    b.table = np.full((1, b.max_pages), -1, np.int32)
    b.table[0, -2:] = [1, 0]
    q, k, v = (b.rng.standard_normal((b.tokens, n * D)).astype(F32) for n in (H, G, G))
    log(f"positions from {first} {news} {dtype.__name__}")
    d = desc_of(b, H, local_window_size=window)
    lens = [dev(x) for x in (b.cu, b.past, b.table)]
    src, qo, kc, vc = [dev(x) for x in (q, k, v)], torch.empty(b.tokens, H * D, device="cuda"), dev(b.k), dev(b.v)
    native.paged_append(d, *map(ptr, src), None, None, *map(ptr, lens), None, None, ptr(qo), ptr(kc), ptr(vc), stream())
    want = b.k.copy(), b.v.copy()
    for t, r, pos in b.each_token():
        for w, x in zip(want, (k, v)):
            w.reshape(-1, G, D)[b.row(r, pos)] = x[t].reshape(G, D)
    assert np.array_equal(host(kc), want[0]) and np.array_equal(host(vc), want[1])
    b.k, b.v = want
    n = native.paged_attention_workspace_size(d)
    ws, out = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), torch.empty_like(qo)
    native.paged_attention(d, ptr(qo), *map(ptr, lens), ptr(kc), ptr(vc), ptr(out), ptr(ws), n, stream())
    check_attention(host(out), b, q, H, window)


def test_positions_without_a_page_are_dropped(gpu):
    """From 2^31 - 4096 on there is no page, whatever the table holds."""
    import torch
    H, G, D, page, first = 2, 1, 64, 1 << 16, 2 ** 31 - 4096 - 3
    b = ref.Batch(107, [8], [1], G, D, page, F32)
    b.max_pages = 1 << 15
    b.table = np.zeros((1, b.max_pages), np.int32)
    d = desc_of(b, H)
    q, k, v = (dev(b.rng.standard_normal((8, n * D)).astype(F32)) for n in (H, G, G))
    kc, vc = dev(b.k), dev(b.v)
    lens = [dev(x) for x in (b.cu, np.array([first], np.int32), b.table)]
    log("positions past the last")
    native.paged_append(d, ptr(q), ptr(k), ptr(v), None, None, *map(ptr, lens), None, None, ptr(torch.empty_like(q)), ptr(kc),
                        ptr(vc), stream())
    want = b.k.copy()
    want.reshape(-1, G, D)[first % page:first % page + 3] = host(k)[:3].reshape(3, G, D)
    assert np.array_equal(host(kc), want)


# news, pasts, H, G, D, page, window: the window's start anywhere in a block of keys
GONE = [
    ([150], [400], 8, 2, 128, 16, 100),
    ([130, 70], [333, 90], 8, 2, 64, 10, 75),
    ([200], [1000], 4, 1, 96, 16, 129),
    ([90, 1], [517, 300], 8, 2, 128, 10, 64),
    ([90], [517], 8, 2, 256, 16, 64),
    ([3, 1], [200, 333], 8, 2, 128, 16, 50),
]


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(GONE)))
def test_pages_behind_a_window_may_be_gone(gpu, case, dtype):
    """With every page wholly before the first new token's window released, the call does the same work:
    the same bits as with the pages there (rows done over for a page that is missing differ)."""
    news, pasts, H, G, D, page, window = GONE[case]
    b = ref.Batch(500 + case, news, pasts, G, D, page, dtype)
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    log(f"pages gone {GONE[case]} {dtype.__name__}")
    there = run_attention(b, q, H, window)
    for r, past in enumerate(pasts):
        b.table[r, :max(0, past - window + 1) // page] = -1
    assert (b.table == -1).any()
    gone = run_attention(b, q, H, window)
    check_attention(gone, b, q, H, window)
    assert np.array_equal(gone, there)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("case", range(len(GONE)))
def test_pages_gone_beside_a_page_of_nans(gpu, case, dtype):
    """What stands for a page that is gone is a row of the request itself, not whatever the cache's first
    page holds (never written, say): the same bits again."""
    news, pasts, H, G, D, page, window = GONE[case]
    b = ref.Batch(500 + case, news, pasts, G, D, page, dtype)
    b.table[b.table >= 0] += 1            # page 0 is nobody's
    b.num_pages += 1
    b.k, b.v = (np.concatenate([np.full_like(x[:1], np.nan), x]) for x in (b.k, b.v))
    q = b.rng.standard_normal((b.tokens, H * D)).astype(F32)
    log(f"pages gone beside NaN {GONE[case]} {dtype.__name__}")
    there = run_attention(b, q, H, window)
    for r, past in enumerate(pasts):
        b.table[r, :max(0, past - window + 1) // page] = -1
    gone = run_attention(b, q, H, window)
    check_attention(gone, b, q, H, window)
    assert np.array_equal(gone, there)
