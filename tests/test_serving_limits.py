"""Host-side tests of the serving-step operators' limits: workspaces, lengths and buffers at the
borders of what the entries take."""
from __future__ import annotations

import pytest

from modelsharp_amd import native

P, MB = 1 << 20, 1 << 20   # addresses that are never followed


def paged(**kw):
    d = dict(tokens=4, requests=2, num_heads=4, kv_num_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4,
             cache_type=native.MS_HIP_DTYPE_F16, local_window_size=-1)
    return native.PagedDesc(**{**d, **kw})


def refused(call, status, words):
    with pytest.raises(native.HipError, match=words) as e:
        call()
    assert e.value.status == status


@pytest.mark.parametrize("size", [-1, -2 ** 31, -2 ** 63])
def test_a_negative_workspace_size_is_no_workspace(size):
    """The keys are not shared out then, so that a workspace inside the cache is not written and
    not refused: the call gets as far as its launch, which a host without a GPU does not have."""
    if native.available():
        pytest.skip("would launch on addresses that nothing lies at")
    d = paged(tokens=1, requests=1, num_pages=4096, max_pages=4096)
    n = native.paged_attention_workspace_size(d)
    assert n > 0
    q, cu, past, table, out, kc, vc = (P + i * 64 * MB for i in range(7))
    refused(lambda: native.paged_attention(d, q, cu, past, table, kc, vc, out, kc, n), 1, "workspace overlaps")
    refused(lambda: native.paged_attention(d, q, cu, past, table, kc, vc, out, kc, size), 3, "launch_paged_attention")
