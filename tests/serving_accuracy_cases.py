"""Inputs of the accuracy tests of paged attention, shared by the GPU tests and by the host tests that
show what those can tell apart."""
from __future__ import annotations

import numpy as np

import serving_ref as ref

# news, pasts, H, G, D, page, window: tiles of 16 rows and of 128, pages of whole and of odd tiles
SHAPES = {
    "tokens-64": ([1, 2, 1], [0, 40, 130], 8, 2, 64, 16, -1),
    "tokens-128": ([1, 1], [70, 200], 8, 2, 128, 10, -1),
    "tokens-256": ([2], [90], 4, 2, 256, 16, -1),
    "chunk-64": ([150], [0], 8, 1, 64, 16, -1),
    "chunk-96": ([70, 61], [20, 0], 8, 2, 96, 10, 60),
    "chunk-128": ([140], [9], 8, 2, 128, 16, -1),
    "chunk-256": ([90], [0], 8, 2, 256, 16, -1),
    "both-128": ([100, 1, 3], [5, 90, 0], 8, 2, 128, 16, -1),
}


def plain(name, dtype):
    """Ordinary values: (batch, queries, heads, window)."""
    news, pasts, H, G, D, page, window = SHAPES[name]
    b = ref.Batch(300 + sorted(SHAPES).index(name), news, pasts, G, D, page, dtype)
    return b, b.rng.standard_normal((b.tokens, H * D)).astype(np.float32), H, window


def small_weights(name, dtype, exponent):
    """Every head's first visible key has a weight near 1 and values near 1e-3, the others weights near
    2^exponent of it and values up to 6e4: rows whose size the small weights' values decide or
    reach. Scores come from two channels of few bits, so that they are exact."""
    news, pasts, H, G, D, page, window = SHAPES[name]
    b = ref.Batch(400 + sorted(SHAPES).index(name), news, pasts, G, D, page, dtype)
    q = np.zeros((b.tokens, H, D), np.float32)
    q[:, :, 0] = 1.0
    q[:, :, 1] = b.rng.integers(-16, 17, (b.tokens, H)) / 16
    b.k[:] = 0.0
    k, v = b.k.reshape(-1, G, D), b.v.reshape(-1, G, D)
    k[:, :, 0] = exponent
    k[:, :, 1] = b.rng.integers(-16, 17, k.shape[:2]) / 16
    v[:] = b.rng.uniform(-6e4, 6e4, v.shape).astype(dtype)
    for r in range(len(b.news)):
        for j in range(b.pasts[r] + b.news[r]):
            if j % 50 == 0:   # a window sees one of these, or none
                row = b.row(r, j)
                k[row, :, :2] = 0.0
                v[row] = b.rng.uniform(-1e-3, 1e-3, v[row].shape).astype(dtype)
    return b, q.reshape(b.tokens, H * D), H, window


LN2 = float(np.log(2.0))   # scores are in powers of two: a scale of ln 2


def wide_queries(name, dtype):
    """Queries with a channel 2^30 times the others, at which no key has a value."""
    b, q, H, window = plain(name, dtype)
    q.reshape(b.tokens, H, b.D)[:, :, 3] *= np.float32(2.0 ** 30)
    b.k[..., 3] = 0.0
    return b, q, H, window


def relative(got, b, q, H, window, scale=0.0):
    """Errors of every output relative to its own sum of w |v|."""
    want, sums, _, _ = ref.attention_sums(b, q, H, window, scale)
    rows = np.array([t for t, _, _ in b.each_token()], int)
    return (np.abs(got.reshape(want.shape)[rows] - want[rows]) / sums[rows]).reshape(-1)


def worst(got, b, q, H, window, scale=0.0, exact_scores=False):
    """The largest error, as a share of attention_own_tolerance."""
    want, sums, mass, keys = ref.attention_sums(b, q, H, window, scale)
    rows = np.array([t for t, _, _ in b.each_token()], int)
    tol = ref.attention_own_tolerance(sums, mass, keys, b.D, exact_scores)
    return float((np.abs(got.reshape(want.shape)[rows] - want[rows]) / tol[rows]).max())


def rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


# A plain float32 evaluation rounds each operand, product and weight by up to EPS24; the kernels' forms
# by up to 2 (fp16 halves) and 8 of it (six bf16 products), beside the same sums.
RMS_FACTOR = 8.0
