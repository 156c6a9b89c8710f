"""Plain 64-bit forms of the serving-step operators (paged append, paged attention, query and key
norms with rotation, low-rank adapters), and seeded inputs for them. numpy on the host."""
from __future__ import annotations

import math

import numpy as np

EPS24 = 2.0 ** -24   # half a step of fp32, relative


class Batch:
    """A ragged batch over a paged cache: lengths, page table (pages in any order), cache of
    `dtype` filled with normal values."""

    def __init__(self, seed, news, pasts, G, D, page, dtype, spare_pages=2, spare_rows=0, extra_columns=0):
        rng = np.random.default_rng(seed)
        self.rng, self.news, self.pasts, self.G, self.D, self.page = rng, list(news), list(pasts), G, D, page
        need = [-(-(n + p) // page) for n, p in zip(news, pasts)]
        self.num_pages = sum(need) + spare_pages
        self.max_pages = max(need + [1]) + extra_columns
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((len(news), self.max_pages), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.past = np.asarray(pasts, np.int32)
        self.tokens = int(self.cu[-1]) + spare_rows
        shape = (self.num_pages, page, G, D)
        self.k = rng.standard_normal(shape).astype(dtype)
        self.v = rng.standard_normal(shape).astype(dtype)

    def row(self, r, pos):
        """The cache row of a position, or -1."""
        pg = pos // self.page
        if pg >= self.max_pages:
            return -1
        e = int(self.table[r, pg])
        return e * self.page + pos % self.page if 0 <= e < self.num_pages else -1

    def each_token(self):
        """(row of the step's tensors, request, position) of every token."""
        for r, (n, p) in enumerate(zip(self.news, self.pasts)):
            for i in range(n):
                yield int(self.cu[r]) + i, r, p + i


def attention(b: Batch, q, H, window=-1, scale=0.0, out=None):
    """(out [tokens, H * D] in 64 bits, largest sum |q| |k| scale, longest range of keys). Rows of no
    request keep `out`."""
    G, D = b.G, b.D
    scale = scale or 1.0 / math.sqrt(D)
    k, v = b.k.reshape(-1, G, D).astype(np.float64), b.v.reshape(-1, G, D).astype(np.float64)
    q = q.reshape(b.tokens, H, D).astype(np.float64)
    out = np.zeros((b.tokens, H, D)) if out is None else out.reshape(b.tokens, H, D).astype(np.float64)
    mass, longest = 0.0, 1
    for t, r, pos in b.each_token():
        lo = max(0, pos - window + 1) if window >= 0 else 0
        rows = np.array([x for x in (b.row(r, j) for j in range(lo, pos + 1)) if x >= 0], np.int64)
        longest = max(longest, len(rows))
        for h in range(H):
            g = h // (H // G)
            if not len(rows):
                out[t, h] = 0.0
                continue
            with np.errstate(all="ignore"):
                s = k[rows, g] @ q[t, h] * scale
                fin = np.abs(k[rows, g]) @ np.abs(q[t, h]) * abs(scale)
                mass = max(mass, float(np.max(fin, where=np.isfinite(fin), initial=0.0)))
                w = np.exp(s - s.max())
                out[t, h] = (w / w.sum()) @ v[rows, g]
    return out.reshape(b.tokens, H * D), mass, longest


def attention_tolerance(mass, longest, D, v_max):
    """How far fp32 attention may be from 64 bits, absolutely. A score is a sum of D products of
    queries rounded to 22 bits (half a step of those: 4 EPS24) added in fp32 (at most D / 4 + 8
    roundings of a partial sum no larger than mass = sum |q| |k| scale) and scaled (3 roundings), and
    a weight's relative error is its score's absolute one. exp2 and the running maximum's
    rescalings round each weight a few times (8), the sum over n keys adds n / 4 + 32 roundings in
    numerator and denominator (a lane's own keys, then the joins), and both errors count twice,
    once in each."""
    ds = mass * (4 + D / 4 + 8 + 3) * EPS24
    return 2 * v_max * (ds + (8 + longest / 4 + 32) * EPS24)


def normed_rotated(x, gamma, pos, cos, sin, interleaved, eps):
    """x [heads, D] of one token: norm per head (gamma None: none), rotation by row
    min(pos, rows - 1) (cos None: none). 64 bits."""
    x = x.astype(np.float64)
    D = x.shape[-1]
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * gamma.astype(np.float64)
    if cos is None:
        return x
    half = min(2 * cos.shape[1], D) // 2
    j = np.arange(half)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    c, s = (m[min(max(pos, 0), m.shape[0] - 1), :half].astype(np.float64) for m in (cos, sin))
    y = x.copy()
    y[:, a] = x[:, a] * c - x[:, b] * s
    y[:, b] = x[:, b] * c + x[:, a] * s
    return y


def norm_tolerance(D, gamma, x_max, rotated):
    """How far the fp32 norm and rotation may be from 64 bits, absolutely. The sum of D squares
    (D / 8 + 8 roundings), its mean, root and reciprocal (5) give inv to half the first plus the
    rest, x * inv * gamma two more roundings; a rotation adds two products and a sum of values
    no larger than sqrt(2) times the largest (3 roundings of each)."""
    rel = ((D / 8 + 8) / 2 + 5 + 2) * EPS24 if gamma is not None else 0.0
    return x_max * math.sqrt(2) * (rel + (4 * EPS24 if rotated else 0.0)) + 1e-30


def lora(x, a, b, ranks, scales, which, base):
    """(y, largest magnitude of the sums' terms) in 64 bits."""
    y = np.zeros((x.shape[0], b.shape[1])) if base is None else base.astype(np.float64)
    terms = np.zeros_like(y)
    for t, ad in enumerate(which):
        if not 0 <= ad < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else int(np.clip(ranks[ad], 0, a.shape[1]))
        s = 1.0 if scales is None else float(scales[ad])
        A, B, xt = a[ad, :r].astype(np.float64), b[ad, :, :r].astype(np.float64), x[t].astype(np.float64)
        y[t] += s * (B @ (A @ xt))
        terms[t] = abs(s) * (np.abs(B) @ (np.abs(A) @ np.abs(xt)))
    return y, terms


def lora_tolerance(y, terms, K, R):
    """How far the fp32 adapters may be from 64 bits, by element: each of the K + R terms' products
    and partial sums is rounded (at most K / 8 + R / 4 + 24 roundings of a sum no larger than the
    terms' magnitudes: the lanes' chains, the waves' and splits' joins), and the last sum with
    the base."""
    return terms * (K / 8 + R / 4 + 24) * EPS24 + (np.abs(y) + terms) * 2 * EPS24 + 1e-30


# ---- bounds by a row's own size ----------------------------------------------------------------

def attention_sums(b: Batch, q, H, window=-1, scale=0.0):
    """(out, sums, mass, keys), 64 bits, [tokens, H, D] and [tokens, H]: out, the sum of w |v| of each
    output, the largest sum |q| |k| scale of a row's visible keys, and how many it sees. Rows of no
    request are NaN."""
    G, D = b.G, b.D
    scale = scale or 1.0 / math.sqrt(D)
    k, v = b.k.reshape(-1, G, D).astype(np.float64), b.v.reshape(-1, G, D).astype(np.float64)
    q = q.reshape(b.tokens, H, D).astype(np.float64)
    out, sums = np.full((b.tokens, H, D), np.nan), np.full((b.tokens, H, D), np.nan)
    mass, keys = np.zeros((b.tokens, H)), np.zeros((b.tokens, H))
    for t, r, pos in b.each_token():
        lo = max(0, pos - window + 1) if window >= 0 else 0
        rows = np.array([x for x in (b.row(r, j) for j in range(lo, pos + 1)) if x >= 0], np.int64)
        for h in range(H):
            g = h // (H // G)
            s = k[rows, g] @ q[t, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h], sums[t, h] = w @ v[rows, g], w @ np.abs(v[rows, g])
            mass[t, h] = (np.abs(k[rows, g]) @ np.abs(q[t, h])).max() * abs(scale)
            keys[t, h] = len(rows)
    return out, sums, mass, keys


def attention_own_tolerance(sums, mass, keys, D, exact_scores=False):
    """How far attention may be from 64 bits, output by output, relative to its own sum of w |v|. A
    score's operands are held to 8 EPS24 (three bf16 parts with six products; fp16 halves 2), its D
    products added in at most D / 4 + 8 roundings and scaled in 3. A weight is the exponential (2) of
    that, held to 8, and counts in numerator and denominator, whose sums over the keys take at most
    keys / 4 + 16 roundings each. Where operands are of so few bits that products and their sums are
    exact (exact_scores), a score is rounded by its scaling alone."""
    ds = mass * (3 if exact_scores else 8 + D / 4 + 8 + 3)
    return sums * (2 * (ds + 2 + 8 + keys / 4 + 16) * EPS24)[..., None]


def halves(x, exp, low):
    """x as the high and low fp16 halves of x * 2^exp, the low one times 2^low, each in 64 bits and scaled
    back: what the fp16 matrix cores are given."""
    y = np.asarray(x, np.float32).astype(np.float64) * 2.0 ** exp
    hi = y.astype(np.float16).astype(np.float64)
    lo = ((y - hi) * 2.0 ** low).astype(np.float16).astype(np.float64)
    return hi * 2.0 ** -exp, lo * 2.0 ** -(low + exp)


def bf16_parts(x):
    """x as three bf16 parts, each cut."""
    out, rest = [], np.asarray(x, np.float32)
    for _ in range(3):
        p = (rest.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        out.append(p.astype(np.float64))
        rest = (rest - p).astype(np.float32)
    return out


def attention_form(b: Batch, q, H, form, window=-1, scale=0.0):
    """Attention as a form of the kernels' products has it, everything else in 64 bits. form:
    "f32"          plain: float32 throughout
    "halves"       queries and weights as two fp16 halves, the low one times 2^12
    "one scale"    the same with the low half unscaled
    "no low q", "no low w"    without the one or the other low half
    "six", "three"            three bf16 parts of everything, six products, three of them
    [tokens, H, D]; rows of no request are NaN."""
    G, D = b.G, b.D
    scale = scale or 1.0 / math.sqrt(D)
    f32 = form == "f32"
    k, v = (x.reshape(-1, G, D).astype(np.float32) for x in (b.k, b.v))
    q = q.reshape(b.tokens, H, D).astype(np.float32)
    out = np.full((b.tokens, H, D), np.nan)
    low = 0 if form == "one scale" else 12

    def product(a, x, exp, drop):   # a [keys, D] and x: matrix by vector or vector by matrix, in a's order
        if form in ("six", "three"):
            pairs = [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)][0 if form == "six" else 3:]
            pa, px = bf16_parts(a), bf16_parts(x)
            return sum(pa[i] @ px[j] for i, j in pairs)
        hi, lo = halves(x, exp, low)
        return a.astype(np.float64) @ hi + (0.0 if drop else a.astype(np.float64) @ lo)

    for t, r, pos in b.each_token():
        lo_key = max(0, pos - window + 1) if window >= 0 else 0
        rows = np.array([x for x in (b.row(r, j) for j in range(lo_key, pos + 1)) if x >= 0], np.int64)
        for h in range(H):
            kk, vv = k[rows, h // (H // G)], v[rows, h // (H // G)]
            if f32:
                s = (kk @ q[t, h]) * np.float32(scale)
                w = np.exp(s - s.max())
                out[t, h] = (w @ vv) / w.sum(dtype=np.float32)
                continue
            e = 15 - int(np.frexp(np.abs(q[t, h]).max())[1])
            s = product(kk, q[t, h], e, form == "no low q") * scale
            w = np.exp(s - s.max()).astype(np.float32)
            out[t, h] = product(vv.T.copy(), w, 11, form == "no low w") / w.sum(dtype=np.float64)
    return out
