"""Host-side tests of the serving-step operators' limits: workspaces, lengths and buffers at the
borders of what the entries take."""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess

import pytest

from modelsharp_amd import native

CSRC = pathlib.Path(__file__).resolve().parents[1] / "modelsharp_amd" / "csrc"
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


@pytest.mark.parametrize("size", [-1, -2 ** 40])
def test_group_query_attention_takes_a_negative_workspace_size_as_none(size):
    """A history whose scores do not fit one workgroup is refused without a workspace."""
    d = native.GqaDesc(batch=1, q_seq=1, kv_seq=0, past_seq=100000, past_in_present=1, num_heads=2, kv_num_heads=1,
                       head_dim=32, present_capacity=100000, local_window_size=-1)
    n = native.gqa_workspace_size(d)
    assert n > 0
    args = [P + i * 64 * MB for i in range(3)] + [None] * 5 + [P + (8 + i) * 1024 * MB for i in range(4)]
    refused(lambda: native.gqa(d, *args, 0), 4, "history too long")
    refused(lambda: native.gqa(d, *args, size), 4, "history too long")


@pytest.fixture(scope="module")
def lengths(tmp_path_factory):
    """paged_span and paged_tiles of the kernels' own header, compiled for the host: lines of cu[r],
    cu[r + 1], tokens, query heads of a kv head and a tile's rows in; first, count and tiles out."""
    hipcc = shutil.which("hipcc", path="/opt/rocm/bin:" + os.environ.get("PATH", ""))
    if not hipcc:
        pytest.skip("no hipcc")
    at = tmp_path_factory.mktemp("lengths")
    (at / "lengths.hip").write_text("""
#include <cstdio>
#include "serving.h"
int main()
{
    int c0, c1, tokens, grp, bm;
    while (std::scanf("%d %d %d %d %d", &c0, &c1, &tokens, &grp, &bm) == 5) {
        const msnb::PagedSpan s = msnb::paged_span(c0, c1, tokens);
        std::printf("%d %d %d\\n", s.first, s.count, msnb::paged_tiles(s.count * grp, bm));
    }
}
""")
    subprocess.run([hipcc, "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-I", str(CSRC), "-o",
                    str(at / "lengths"), str(at / "lengths.hip")], check=True, capture_output=True)

    def run(rows):
        out = subprocess.run([str(at / "lengths")], input="\n".join(" ".join(map(str, r)) for r in rows), check=True,
                             capture_output=True, text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def test_lengths_that_make_no_sense_are_cut_to_the_tensors_rows(lengths):
    lo, hi = -2 ** 31, 2 ** 31 - 1
    some = [lo, lo + 1, -5, -1, 0, 1, 7, 30, 31, 100, hi - 1, hi]
    rows = [(c0, c1, tokens, 4, bm) for c0 in some for c1 in some for tokens in (1, 30, 2 ** 29) for bm in (16, 128)]
    for (c0, c1, tokens, grp, bm), (first, count, tiles) in zip(rows, lengths(rows)):
        begin = min(max(c0, 0), tokens)
        assert first == begin and count == max(min(c1, tokens) - begin, 0), (c0, c1, tokens)
        assert 0 <= first <= first + count <= tokens
        assert tiles == min(-(-count * grp // bm), 2 ** 24)
    # the most rows that a call may have
    assert lengths([(0, 1, 1, hi, 16), (0, 1, 1, hi, 128)]) == [(0, 1, 2 ** 24), (0, 1, 2 ** 24)]


def test_outputs_do_not_overlap_the_small_inputs():
    """Lengths, tables, norm weights, rotary caches, positions, ranks and scales are inputs too: an output or a
    workspace on them is refused before anything is launched."""
    at = [P + i * 64 * MB for i in range(14)]
    q, k, v, gq, gk, cu, past, table, cos, sin, out, kc, vc, ws = at
    d = paged(do_rotary=1, cos_rows=64, cos_cols=32)
    good = [q, k, v, gq, gk, cu, past, table, cos, sin, out, kc, vc]
    last = {gq: 63, gk: 63, cu: 2, past: 1, table: 2 * 4 - 1, cos: 64 * 32 - 1, sin: 64 * 32 - 1}   # elements
    for i in (10, 11, 12):
        for j in (3, 4, 5, 6, 7, 8, 9):
            for x in (good[j], good[j] + 4 * last[good[j]] & ~15):
                refused(lambda: native.paged_append(d, *[x if n == i else y for n, y in enumerate(good)]), 1, "overlaps")
    d = paged(tokens=1, requests=1, num_pages=4096, max_pages=4096)
    n = native.paged_attention_workspace_size(d)
    assert n > 0
    for x in (cu, past, table, table + 4 * 4092):
        refused(lambda: native.paged_attention(d, q, cu, past, table, kc, vc, x), 1, "overlaps")
        refused(lambda: native.paged_attention(d, q, cu, past, table, kc, vc, out, x, n), 1, "overlaps")
    d = native.QkNormDesc(tokens=4, num_heads=4, kv_num_heads=2, head_dim=64, do_rotary=1, cos_rows=8, cos_cols=32)
    good = [q, k, gq, gk, past, cos, sin, out, kc]
    for i in (7, 8):
        for j in (2, 3, 4, 5, 6):
            refused(lambda: native.qk_norm_rotary(d, *[good[j] if n == i else y for n, y in enumerate(good)]), 1, "overlaps")
    d = native.LoraDesc(tokens=4, K=64, N=32, adapters=2, max_rank=8, weight_type=native.MS_HIP_DTYPE_F16)
    n = native.lora_workspace_size(d)
    good = [q, k, v, gq, gk, cu, past, out, ws]   # x, a, b, ranks, scales, which, base, y, workspace
    for i in (7, 8):
        for j in (3, 4, 5):
            refused(lambda: native.lora(d, *[good[j] if m == i else y for m, y in enumerate(good)], n), 1, "overlaps")
