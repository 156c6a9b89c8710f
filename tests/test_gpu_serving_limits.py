"""The serving-step operators on the GPU at the borders of what their entries take: workspaces,
lengths, pages that are not there."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from modelsharp_amd import native
from test_gpu_serving import F16, F32, check_attention, desc_of, dev, host, log, ptr, stream

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
