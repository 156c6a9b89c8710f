"""What the accuracy tests of paged attention can tell apart, on the host: the kernels' forms of the
products stay inside their bounds, forms with fewer bits do not."""
from __future__ import annotations

import numpy as np
import pytest

import serving_accuracy_cases as cases
import serving_ref as ref

F16, F32 = np.float16, np.float32


@pytest.mark.parametrize("name", sorted(cases.SHAPES))
def test_ordinary_values_tell_the_forms_apart(name):
    for dtype, good, bad in ((F16, "halves", ("no low q", "no low w")), (F32, "six", ("three",))):
        b, q, H, window = cases.plain(name, dtype)
        plain = cases.rms(cases.relative(ref.attention_form(b, q, H, "f32", window), b, q, H, window))
        got = ref.attention_form(b, q, H, good, window)
        assert cases.worst(got, b, q, H, window) <= 1
        assert cases.rms(cases.relative(got, b, q, H, window)) <= cases.RMS_FACTOR * plain
        for form in bad:
            assert cases.rms(cases.relative(ref.attention_form(b, q, H, form, window), b, q, H, window)) > \
                3 * cases.RMS_FACTOR * plain, (form, dtype)


@pytest.mark.parametrize("exponent", [-30, -20])
@pytest.mark.parametrize("name", ["tokens-64", "chunk-64", "chunk-128"])
def test_small_weights_beside_larger_values(name, exponent):
    b, q, H, window = cases.small_weights(name, F16, exponent)
    good, bad = (cases.worst(ref.attention_form(b, q, H, form, window, cases.LN2), b, q, H, window, cases.LN2, True)
                 for form in ("halves", "one scale"))
    assert good <= 1
    if exponent == -30:   # (2^-20: off by 2e-6 of a row, which the bound's sums leave room for)
        assert bad > 10


@pytest.mark.parametrize("name", ["tokens-64", "chunk-64"])
def test_queries_with_one_large_channel(name):
    b, q, H, window = cases.wide_queries(name, F16)
    assert cases.worst(ref.attention_form(b, q, H, "halves", window), b, q, H, window) <= 1
    assert cases.worst(ref.attention_form(b, q, H, "one scale", window), b, q, H, window) > 10
