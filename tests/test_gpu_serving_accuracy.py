"""Paged attention on the GPU by each output's own size: ordinary values, small weights beside larger
values, queries of a wide range."""
from __future__ import annotations

import numpy as np
import pytest

import serving_accuracy_cases as cases
import serving_ref as ref
from test_gpu_serving import F16, F32, log, lora_inputs, run_attention, run_lora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("workspace", [True, False], ids=["split", "whole"])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("name", sorted(cases.SHAPES))
def test_ordinary_values(gpu, name, dtype, workspace):
    b, q, H, window = cases.plain(name, dtype)
    plain = cases.rms(cases.relative(ref.attention_form(b, q, H, "f32", window), b, q, H, window))
    got = run_attention(b, q, H, window, workspace=workspace)
    share, err = cases.worst(got, b, q, H, window), cases.rms(cases.relative(got, b, q, H, window))
    log(f"ordinary {name} {dtype.__name__}: {share:.3f} of the bound, rms {err:.2e}, float32 {plain:.2e}")
    assert share <= 1 and err <= cases.RMS_FACTOR * plain


@pytest.mark.parametrize("workspace", [True, False], ids=["split", "whole"])
@pytest.mark.parametrize("exponent", [-30, -20])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("name", [n for n in sorted(cases.SHAPES) if n != "chunk-96"])
def test_small_weights_beside_larger_values(gpu, name, dtype, exponent, workspace):
    b, q, H, window = cases.small_weights(name, dtype, exponent)
    got = run_attention(b, q, H, window, scale=cases.LN2, workspace=workspace)
    share = cases.worst(got, b, q, H, window, cases.LN2, True)
    log(f"small weights {name} {dtype.__name__} 2^{exponent}: {share:.3f} of the bound")
    assert share <= 1


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("name", sorted(cases.SHAPES))
def test_queries_with_one_large_channel(gpu, name, dtype):
    b, q, H, window = cases.wide_queries(name, dtype)
    share = cases.worst(run_attention(b, q, H, window), b, q, H, window)
    log(f"wide queries {name} {dtype.__name__}: {share:.3f} of the bound")
    assert share <= 1


@pytest.mark.parametrize("T,R", [(5, 16), (40, 24), (40, 64), (200, 130), (640, 16), (640, 64)])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_adapters_whose_ranks_differ_widely(gpu, dtype, T, R):
    """One rank 2^30 times the others, which no output takes: the others keep their bits."""
    case = (T, 256, 264, 3, R, "mixed", False, "new")
    x, a, b, ranks, scales, which, y0 = lora_inputs(case, dtype, 47)
    x[:, 0] = F32(2.0 ** 30)
    a[:, :, 0] = 0.0
    a[:, 3, 0] = 1.0
    b[:, :, 3] = 0.0
    want, terms = ref.lora(x, a, b, ranks, scales, which, y0)
    got = run_lora(case, x, a, b, ranks, scales, which, y0, False)
    share = np.max(np.abs(got - want) / ref.lora_tolerance(want, terms, 256, R))
    log(f"wide ranks {T} {R} {dtype.__name__}: {share:.3f} of the bound")
    assert share <= 1
