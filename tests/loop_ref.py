"""Plain forms of what a server's loop needs around a step (plan and commit, sampling), and seeded inputs
for them. numpy on the host, 64 bits."""
from __future__ import annotations

import math

import numpy as np

POSITIONS = 2 ** 31 - 4096   # positions from here on have no page


def ceil(a, b):
    return -(-a // b)


def plan(want, past, free, count, table, tokens, page, num_pages):
    """(cu, used, request, position, slot, table) of a step, one request after the other."""
    want, past, free, table = (np.asarray(x).astype(np.int64) for x in (want, past, free, table))
    table, width, count = table.copy(), table.shape[1], int(np.clip(count, 0, num_pages))
    cu, rows, used, asked, wanted = [0], [], 0, 0, 0
    for r, (w, p) in enumerate(zip(want, np.maximum(past, 0))):
        served = 0
        if w > 0 and p + w <= POSITIONS and ceil(p + w, page) <= width:
            need = ceil(p + w, page) - ceil(p, page)
            asked, wanted = asked + w, wanted + need
            if asked <= tokens and (need == 0 or wanted <= count):
                served = int(w)
                for col in range(ceil(p, page), ceil(p + w, page)):
                    table[r, col] = free[count - 1 - used]
                    used += 1
        for pos in range(p, p + served):
            e = table[r, pos // page]
            rows.append((r, pos, e * page + pos % page if 0 <= e < num_pages else -1))
        cu.append(cu[-1] + served)
    rows += [(-1, -1, -1)] * (tokens - len(rows))
    request, position, slot = np.array(rows, np.int64).reshape(-1, 3).T
    return tuple(np.asarray(x, np.int64) for x in (cu, used, request, position, slot, table))


def commit(cu, used, done, keep, past, table, free, count, page, num_pages):
    """(past, table, free, count) behind a step."""
    cu, past, table, free = (np.asarray(x).astype(np.int64).copy() for x in (cu, past, table, free))
    count = int(np.clip(count, 0, num_pages))
    count -= int(np.clip(used, 0, count))
    for r in range(len(past)):
        after = min(max(past[r], 0) + max(cu[r + 1] - cu[r], 0), POSITIONS)
        past[r] = after
        if done is not None and done[r]:
            past[r] = 0
            first = 0 if keep is None else max(int(keep[r]), 0)
            for col in range(first, min(ceil(after, page), table.shape[1])):
                e = table[r, col]
                table[r, col] = -1
                if 0 <= e < num_pages and count < num_pages:
                    free[count] = e
                    count += 1
    return past, table, free, count


class Pool:
    """Requests over a pool of pages in any order, with a stack of free ones."""

    def __init__(self, seed, pasts, page, spare, width):
        rng = np.random.default_rng(seed)
        need = [ceil(max(p, 0), page) for p in pasts]
        self.num_pages, self.page = sum(need) + spare, page
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((len(pasts), width), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :min(n, width)] = order[at:at + min(n, width)]
            at += n
        self.free = np.full(self.num_pages, -7, np.int32)
        self.free[:spare] = order[at:]
        self.count = spare
        self.past = np.asarray(pasts, np.int32)
        self.rng = rng


def weights(row, t):
    """(weights, order) of a row of logits in 64 bits: NaN as -infinity, the order by falling logits, ties by
    index. None where there is nothing to draw from."""
    l = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    top = l.max()
    if top == -np.inf:
        return None
    with np.errstate(all="ignore"):
        if not t > 0:
            w = np.zeros(len(l))
            w[int(np.argmax(l))] = 1.0
        else:
            w = np.where(l == top, 1.0, np.exp((l - top) / np.float64(t)))
            w = np.where((l == -np.inf) | np.isnan(w), 0.0, w)
    return w, np.lexsort((np.arange(len(l)), -l))


def sample(row, t=1.0, k=0, p=1.0, m=0.0, u=0.0):
    """(token, logprob, how far the logprob may be off): the definition, and a tolerance from weights that are
    multiples of 2^-frac (off by half of that each, or 2^-45 of their own size) and a result in fp32."""
    found = weights(row, t)
    if found is None:
        return -1, math.nan, 0.0
    w, order = found
    n = len(row)
    if t > 0 and 0 < k < n:
        n = k
    sums = np.cumsum(w[order[:n]])
    if t > 0 and p < 1:
        n = min(n, int(np.searchsorted(sums, max(float(p), 0.0) * sums[-1], side="left")) + 1)
    if t > 0 and m > 0:
        n = max(1, min(n, int((w[order[:n]] >= min(float(m), 1.0)).sum())))
    left = np.sort(order[:n])
    left = left[w[left] > 0]
    sums = np.cumsum(w[left])
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(left) - 1)
    token, total = int(left[at]), sums[-1]
    bits = max(1, (len(row) - 1)).bit_length()
    step = 2.0 ** -(44 if bits < 18 else 62 - bits)
    lp = math.log(w[token] / total)
    off = (step / 2 + w[token] * 2.0 ** -45) / w[token] + (len(left) * step / 2 + total * 2.0 ** -45) / total
    return token, lp, abs(lp) * 2.0 ** -24 + 2 * off


def near_a_border(row, t=1.0, k=0, p=1.0, m=0.0, u=0.0, rel=1e-10):
    """Whether a limit lies within `rel` of a sum or weight it is compared with, so that 64-bit roundings may
    decide (the inputs of a test are chosen so that none does)."""
    found = weights(row, t)
    if found is None or not t > 0:
        return False
    w, order = found
    n = k if 0 < k < len(row) else len(row)
    sums = np.cumsum(w[order[:n]])
    near = False
    if 0 < p < 1:
        near |= bool((np.abs(sums - float(p) * sums[-1]) < rel * sums[-1]).any())
        n = min(n, int(np.searchsorted(sums, float(p) * sums[-1], side="left")) + 1)
    if 0 < m < 1:
        near |= bool((np.abs(w - float(m)) < rel).any())
        n = max(1, min(n, int((w[order[:n]] >= float(m)).sum())))
    left = np.sort(order[:n])
    sums = np.cumsum(w[left])
    if 0 < u < 1:
        near |= bool((np.abs(sums - float(u) * sums[-1]) < rel * sums[-1])[w[left] > 0].any())
    return near
