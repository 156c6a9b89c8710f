"""What a server's loop needs around a step (plan and commit, sampling) on the GPU against plain forms."""
from __future__ import annotations

import numpy as np
import pytest

import loop_ref as ref
from modelsharp_amd import native

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
GUARD = -99


def log(msg):
    print(msg, flush=True)


def dev(x, guard=0):
    """x on the device, `guard` cells behind it."""
    import torch
    if x is None:
        return None
    x = np.ascontiguousarray(x)
    if guard:
        x = np.concatenate([x.reshape(-1), np.full(guard, GUARD, x.dtype)])
    return torch.from_numpy(x).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def unguarded(t, shape):
    """The host copy of a guarded buffer; what lies behind it is as it was."""
    x = t.cpu().numpy()
    n = int(np.prod(shape))
    assert (x[n:] == GUARD).all()
    return x[:n].reshape(shape)


# ---- plan and commit -----------------------------------------------------------------------------

def run_plan(pool, want, tokens, count=None):
    import torch
    R, W = pool.table.shape
    d = native.StepDesc(tokens=tokens, requests=R, page_size=pool.page, num_pages=pool.num_pages, max_pages=W)
    count = pool.count if count is None else count
    ins = [dev(np.asarray(x, I32)) for x in (want, pool.past, pool.free, [count])]
    outs = [dev(x, 5) for x in (pool.table, np.full(R + 1, GUARD, I32), np.full(1, GUARD, I32),
                                *[np.full(tokens, GUARD, I32)] * 3)]
    native.paged_plan(d, *map(ptr, ins), *map(ptr, outs), stream())
    torch.cuda.synchronize()
    table, cu, used, request, position, slot = (unguarded(t, s) for t, s in zip(
        outs, (pool.table.shape, (R + 1,), (), (tokens,), (tokens,), (tokens,))))
    expected = ref.plan(want, pool.past, pool.free, count, pool.table, tokens, pool.page, pool.num_pages)
    for name, got, exp in zip(("cu", "used", "request", "position", "slot", "table"),
                              (cu, used, request, position, slot, table), expected):
        assert np.array_equal(got, exp), name
    for t, x in zip(ins, (want, pool.past, pool.free, [count])):
        assert np.array_equal(t.cpu().numpy(), np.asarray(x))   # a plan can be made again
    return cu, int(used), table


def run_commit(pool, table, cu, used, done, keep, count=None):
    import torch
    R, W = table.shape
    d = native.StepDesc(tokens=int(max(cu.max(), 0)), requests=R, page_size=pool.page, num_pages=pool.num_pages, max_pages=W)
    count = pool.count if count is None else count
    ins = [dev(x) for x in (np.asarray(cu, I32), np.asarray([used], I32), done, keep)]
    outs = [dev(np.asarray(x, I32), 5) for x in (pool.past, table, pool.free, [count])]
    native.paged_commit(d, *map(ptr, ins), *map(ptr, outs), stream())
    torch.cuda.synchronize()
    got = [unguarded(t, s) for t, s in zip(outs, ((R,), table.shape, (pool.num_pages,), ()))]
    expected = ref.commit(cu, used, done, keep, pool.past, table, pool.free, count, pool.page, pool.num_pages)
    for name, g, e in zip(("past", "table", "free", "count"), got, expected):
        assert np.array_equal(g, e), name
    return got


# requests, largest want, largest past, page, spare pages (of what is needed), rows (of what is wanted)
PLANS = [
    (1, 1, 0, 1, 1.0, 1.0), (1, 1, 15, 16, 1.0, 1.0), (1, 40, 16, 16, 1.0, 1.0), (3, 5, 20, 8, 1.0, 2.0),
    (64, 1, 300, 16, 1.0, 1.0), (65, 30, 100, 10, 0.5, 1.0), (200, 50, 0, 24, 1.0, 0.6), (256, 3, 500, 16, 0.3, 0.9),
    (257, 17, 90, 7, 0.8, 0.8), (1024, 2, 40, 16, 1.0, 1.0), (1025, 9, 33, 5, 0.7, 0.7), (2500, 4, 64, 16, 0.9, 1.0),
    (8192, 3, 10, 16, 0.95, 0.95), (40, 900, 2000, 128, 1.0, 1.0), (5, 1, 100, 16, 0.0, 1.0), (6, 20, 50, 16, 1.0, 0.0),
]


@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan_and_commit(gpu, case):
    R, want, past, page, spare, room = PLANS[case]
    log(f"plan {PLANS[case]}")
    rng = np.random.default_rng(case)
    pasts, wants = rng.integers(0, past + 1, R), rng.integers(0 if R > 2 else want, want + 1, R)
    need = sum(ref.ceil(p + w, page) - ref.ceil(p, page) for p, w in zip(pasts, wants))
    width = max(ref.ceil(p + w, page) for p, w in zip(pasts, wants)) + case % 3
    pool = ref.Pool(case, pasts, page, int(need * spare), max(1, width))
    cu, used, table = run_plan(pool, wants, int(sum(wants) * room) + case % 4)
    done = rng.integers(0, 2, R).astype(I32)
    keep = rng.integers(0, 3, R).astype(I32)
    run_commit(pool, table, cu, used, None, None)
    run_commit(pool, table, cu, used, done, None)
    run_commit(pool, table, cu, used, done, keep)
    run_commit(pool, table, cu, used, np.full(R, -1, I32), keep)


def test_plan_of_nothing(gpu):
    pool = ref.Pool(1, [], 16, 4, 3)
    log("no requests")
    run_plan(pool, [], 6)
    run_plan(pool, [], 0)
    pool = ref.Pool(2, [5, 0, 33], 16, 4, 3)
    cu, used, table = run_plan(pool, [0, 0, 0], 7)
    assert used == 0 and not cu.any()
    run_plan(pool, [1, 1, 1], 0)
    pool = ref.Pool(3, [0, 0], 16, 4, 0)   # a table without columns
    run_plan(pool, [1, 2], 3)


def test_plan_lengths_that_make_no_sense(gpu):
    """Negative ones, wants that pass the table, the positions or 32 bits in sum: those requests wait, the others are
    served; counts outside the stack are cut to it."""
    big = 2 ** 31 - 1
    pool = ref.Pool(4, [5, -3, 7, 40, 0, 16], 16, 9, 4)
    for want in ([1, 2, -5, 3, 0, 1], [big, 1, 1, 1, 1, 1], [1, big, big, big, big, 2], [-big - 1] * 6, [64, 1, 1, 1, 1, 1],
                 [59, 1, 1, 1, 1, 1], [60, 1, 1, 1, 1, 1]):
        for tokens in (3, 100):
            log(f"want {want} tokens {tokens}")
            run_plan(pool, want, tokens)
    for count in (-1, 0, 1, pool.num_pages, pool.num_pages + 5, big):
        log(f"count {count}")
        cu, used, table = run_plan(pool, [1, 20, 17, 1, 30, 1], 90, count)
        run_commit(pool, table, cu, used, np.ones(6, I32), None, count)
        run_commit(pool, table, cu, big, np.ones(6, I32), None, count)
        run_commit(pool, table, cu, -4, np.ones(6, I32), None, count)
    pool.past[:] = big
    run_plan(pool, [1] * 6, 10)
    run_commit(pool, pool.table, np.arange(7), 0, np.ones(6, I32), np.array([0, 1, 2, -5, 9, big], I32))


def test_what_waits_is_not_passed(gpu):
    """A want above the step's rows holds back all behind it; one whose pages are not free those that need a page."""
    pool = ref.Pool(8, [5, 16, 3, 32, 7], 16, 2, 4)
    for want, tokens, served in (([9, 1, 1, 1, 1], 8, [0, 0, 0, 0, 0]), ([1, 9, 1, 1, 1], 8, [1, 0, 0, 0, 0]),
                                 # 5 + 40 fill 3 pages of 16, 2 of them new and both free; 5 + 50 need 3
                                 ([40, 1, 1, 1, 1], 60, [40, 0, 1, 0, 1]), ([50, 1, 1, 1, 1], 60, [0, 0, 1, 0, 1]),
                                 ([8, 1, 1, 1, 1], 8, [8, 0, 0, 0, 0])):
        log(f"want {want} of {tokens}")
        assert np.diff(run_plan(pool, want, tokens)[0]).tolist() == served


def test_pages_that_are_not_there(gpu):
    """Table and stack entries outside the pool: their rows have no slot and nothing returns them."""
    pool = ref.Pool(5, [40, 20, 70, 1], 16, 12, 6)
    pool.table[0, 1], pool.table[2, 4], pool.free[3], pool.free[11] = -1, pool.num_pages, pool.num_pages + 9, -4
    log("missing pages")
    cu, used, table = run_plan(pool, [20, 30, 12, 50], 112)
    assert used
    for done in ([1, 1, 1, 1], [0, 1, 0, 1], [1, 0, 1, 0]):
        run_commit(pool, table, cu, used, np.array(done, I32), None)


def test_a_page_returned_twice_stays_in_the_stack(gpu):
    pool = ref.Pool(6, [64, 64], 16, 6, 4)
    pool.table[1] = pool.table[0]
    pool.free[:] = np.arange(pool.num_pages)
    log("returned twice")
    run_commit(pool, pool.table, np.zeros(3, I32), 0, np.ones(2, I32), None, pool.num_pages - 3)


def test_plan_replayed_from_a_graph(gpu):
    """Plan and commit captured once; the lengths of each replay are read on the device."""
    import torch
    R, page, W, tokens = 20, 16, 8, 60
    pool = ref.Pool(7, [0] * R, page, 70, W)
    d = native.StepDesc(tokens=tokens, requests=R, page_size=page, num_pages=pool.num_pages, max_pages=W)
    want, past, free, count, table, done = (dev(np.asarray(x, I32)) for x in (
        np.zeros(R), pool.past, pool.free, [pool.count], pool.table, np.zeros(R)))
    cu, used = dev(np.zeros(R + 1, I32)), dev(np.zeros(1, I32))
    rows = [dev(np.zeros(tokens, I32)) for _ in range(3)]

    def step(st):
        native.paged_plan(d, *map(ptr, (want, past, free, count, table, cu, used, *rows)), st)
        native.paged_commit(d, *map(ptr, (cu, used, done)), None, *map(ptr, (past, table, free, count)), st)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(side.cuda_stream)   # nothing is wanted: nothing changes
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step(side.cuda_stream)
    state = [pool.past, pool.table, pool.free, pool.count]
    for i in range(12):
        w, e = pool.rng.integers(0, 6, R).astype(I32), (pool.rng.random(R) < 0.2).astype(I32)
        want.copy_(dev(w))
        done.copy_(dev(e))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        exp = ref.plan(w, state[0], state[2], state[3], state[1], tokens, page, pool.num_pages)
        state = list(ref.commit(exp[0], exp[1], e, None, state[0], exp[5], state[2], state[3], page, pool.num_pages))
        log(f"replay {i}: {exp[0][-1]} rows, {exp[1]} pages, {state[3]} free")
        for name, got, x in zip(("cu", "used", "request", "position", "slot", "past", "table", "free", "count"),
                                (cu, used, *rows, past, table, free, count), (*exp[:5], *state)):
            assert np.array_equal(got.cpu().numpy().reshape(np.shape(x)), x), name


# ---- sampling ------------------------------------------------------------------------------------

def run_sample(logits, t=None, k=None, p=None, m=None, u=None, stride=0, logprobs=True):
    """(tokens, logprobs) of numpy rows."""
    import torch
    rows, vocab = logits.shape
    if stride:
        x = np.full((rows, stride), 1e30, F32)   # what lies between the rows would be drawn
        x[:, :vocab] = logits
    else:
        x = logits
    x = dev(x)
    d = native.SampleDesc(rows=rows, vocab=vocab, stride=stride)
    n = native.sample_workspace_size(d)
    ws = torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    token, lp = dev(np.full(rows, GUARD, I32), 3), dev(np.full(rows, GUARD, F32), 3)
    arrays = [dev(None if a is None else np.asarray(a, ty)) for a, ty in ((t, F32), (k, I32), (p, F32), (m, F32), (u, F32))]
    native.sample(d, ptr(x), *map(ptr, arrays), ptr(token), ptr(lp) if logprobs else None, ptr(ws), n, stream())
    torch.cuda.synchronize()
    assert (ws[n:] == 0xA5).all()
    if not logprobs:
        assert (lp == GUARD).all()
    return unguarded(token, (rows,)), unguarded(lp, (rows,))


def check_sample(logits, t=None, k=None, p=None, m=None, u=None, stride=0):
    rows = logits.shape[0]
    each = [np.full(rows, off) if a is None else np.asarray(a, ty) for a, off, ty in
            ((t, 1.0, F32), (k, 0, I32), (p, 1.0, F32), (m, 0.0, F32), (u, 0.0, F32))]
    for r in range(rows):
        assert not ref.near_a_border(logits[r], *(a[r] for a in each)), r
    token, lp = run_sample(logits, t, k, p, m, u, stride)
    for r in range(rows):
        exp, elp, tol = ref.sample(logits[r], *(a[r] for a in each))
        assert token[r] == exp, (r, token[r], exp, [a[r] for a in each])
        assert (np.isnan(lp[r]) and np.isnan(elp)) or abs(lp[r] - elp) <= tol, (r, lp[r], elp, tol)
    return token


def settings(rng, rows):
    """A mix of settings, some of them off."""
    t = rng.uniform(0.3, 2.0, rows).astype(F32)
    k = np.where(rng.random(rows) < 0.5, rng.integers(1, 300, rows), 0).astype(I32)
    p = np.where(rng.random(rows) < 0.6, rng.uniform(0.05, 0.999, rows), 1.0).astype(F32)
    m = np.where(rng.random(rows) < 0.4, rng.uniform(0.001, 0.3, rows), 0.0).astype(F32)
    t[rng.random(rows) < 0.1] = 0.0
    return dict(t=t, k=k, p=p, m=m, u=rng.random(rows).astype(F32))


VOCABS = [1, 2, 3, 63, 64, 65, 255, 256, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 12289, 32000, 50001, 151936, 270001]


@pytest.mark.parametrize("vocab", VOCABS)
def test_sample(gpu, vocab):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 20000 else 9
    log(f"sample {rows} x {vocab}")
    logits = (rng.standard_normal((rows, vocab)) * 2.5).astype(F32)
    check_sample(logits, **settings(rng, rows), stride=vocab + vocab % 7 if vocab % 2 else 0)
    check_sample(logits, u=rng.random(rows))                                    # no settings at all
    check_sample(logits, p=rng.uniform(0.5, 1.0, rows), u=rng.random(rows))
    check_sample(logits, k=rng.integers(1, vocab + 3, rows), u=rng.random(rows))


@pytest.mark.parametrize("rows", [1, 2, 7, 65, 300])
def test_sample_rows(gpu, rows):
    rng = np.random.default_rng(rows)
    for vocab in (500, 5000):
        log(f"rows {rows} x {vocab}")
        check_sample((rng.standard_normal((rows, vocab)) * 3 + 7).astype(F32), **settings(rng, rows))


@pytest.mark.parametrize("kind", ["equal", "two", "coarse", "steps", "wide", "tiny", "large", "spike", "offset", "zeros"])
def test_sample_distributions(gpu, kind):
    """Ties (by rising index), logits far from 1, differences below a weight's step."""
    rng = np.random.default_rng(3)
    rows, vocab = 16, 30011
    x = rng.standard_normal((rows, vocab))
    logits = {"equal": np.full((rows, vocab), 3.5), "two": np.where(x > 2, 1.0, 0.0), "coarse": np.round(x * 8) / 4,
              "steps": np.round(x * 2), "wide": x * 30, "tiny": x * 1e-30, "large": x * 1e30, "spike": x * 0.1 + (x > 4) * 50,
              "offset": x - 1e4, "zeros": np.where(x > 0, 0.0, -0.0)}[kind].astype(F32)
    log(f"distribution {kind}")
    s = settings(rng, rows)
    if kind == "equal" or kind == "tiny" or kind == "zeros":   # sums of whole numbers: keep off their borders
        s["p"] = np.where(s["p"] < 1, np.round(s["p"] * vocab) / vocab + 0.4 / vocab, 1.0)
        s["u"] = (np.floor(s["u"] * 1000) + 0.37) / 1000
    if kind == "tiny":
        s["m"] = None   # every weight is within a step of the largest
    if kind == "large":
        s["t"] = None
    check_sample(logits, **s)


@pytest.mark.parametrize("vocab", [7, 5000, 50001])
def test_sample_limits(gpu, vocab):
    """Every setting at and past its ends."""
    rng = np.random.default_rng(vocab)
    nan, inf = np.nan, np.inf
    base = (rng.standard_normal(vocab) * 2).astype(F32)
    cases = [dict(t=x) for x in (0.0, -1.0, nan, inf, 1e-30, 1e30, 1e-3, 100.0)]
    cases += [dict(k=x) for x in (-5, 0, 1, 2, vocab - 1, vocab, vocab + 1, 2 ** 31 - 1)]
    cases += [dict(p=x) for x in (-1.0, 0.0, 1e-30, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, inf, nan)]
    cases += [dict(m=x) for x in (-1.0, 0.0, 1e-30, 0.02, 1.0, 2.0, inf, nan)]
    cases += [dict(u=x) for x in (-1.0, 0.0, 1e-30, 1 - 2.0 ** -24, 1.0, 5.0, nan)]
    cases += [dict(t=0.7, k=50, p=0.9, m=0.05), dict(k=1, p=0.0, m=2.0), dict(t=50.0, k=vocab - 1, p=0.99, m=0.9)]
    rows = len(cases)
    log(f"limits at {vocab}")
    off = dict(t=1.0, k=0, p=1.0, m=0.0, u=0.618034)
    # a random number of 1 takes the last token that is left with a weight above zero
    cols = {n: np.array([c.get(n, v) for c in cases], I32 if n == "k" else F32) for n, v in off.items()}
    check_sample(np.tile(base, (rows, 1)), **cols)


@pytest.mark.parametrize("vocab", [5, 4097, 50001])
def test_sample_odd_logits(gpu, vocab):
    """Masked tokens (-infinity, the type's lowest value), NaN, +infinity, nothing at all."""
    rng = np.random.default_rng(vocab)
    low = np.finfo(F32).min
    rows = []
    for odd, share in ((-np.inf, 0.5), (low, 0.5), (np.nan, 0.3), (-np.inf, 0.999), (low, 0.999), (np.inf, 0.3), (-np.inf, 1.0),
                       (np.nan, 1.0), (np.inf, 1.0), (low, 1.0)):
        x = (rng.standard_normal(vocab) * 2).astype(F32)
        x[rng.random(vocab) < share] = odd
        if share < 1:
            x[vocab // 2] = 1.5
        rows.append(x)
    one = np.full(vocab, -np.inf, F32)
    one[vocab - 1] = -2.0
    rows += [one, np.where(np.arange(vocab) == 1, np.inf, np.nan).astype(F32),
             np.where(np.arange(vocab) % 2, np.inf, -np.inf).astype(F32)]
    logits = np.stack(rows)
    n = len(rows)
    log(f"odd logits at {vocab}")
    u = (np.floor(rng.random(n) * 97) + 0.37) / 97
    check_sample(logits, u=u)
    check_sample(logits, t=[0.0] * n, u=u)
    check_sample(logits, p=[0.77] * n, k=[vocab // 2 + 1] * n, m=[0.01] * n, u=u)
    check_sample(logits, k=[2] * n, u=u)


@pytest.mark.parametrize("vocab", [5, 1000, 4097, 8192, 50001])
def test_sample_shares_of_the_lowest_logits(gpu, vocab):
    """Rows whose largest logit is the type's lowest value (or the next above it), by p alone: what is -infinity, NaN or
    behind the row's end has no part in the total that p is a share of."""
    rng = np.random.default_rng(vocab)
    low = np.finfo(F32).min
    next_up = np.nextafter(low, F32(0))
    rows, t = [], []
    for top in (low, next_up):
        for below in ([], [-np.inf], [np.nan], [-np.inf, np.nan], [low], [low, -np.inf]):
            for temperature in (1.0, 0.3, 1e30):   # (at 1e30 `low` weighs e^-20 beside the next above it)
                x = np.full(vocab, top, F32)
                for odd in below:
                    x[rng.random(vocab) < 0.4] = odd
                x[vocab // 2] = top
                rows.append(x)
                t.append(temperature)
    n, logits = len(rows), np.stack(rows)
    log(f"lowest logits at {vocab}")
    for p in (0.0137, 0.43, 0.871):
        u = (np.floor(rng.random(n) * 97) + 0.37) / 97
        check_sample(logits, t=t, p=[p] * n, u=u)
        check_sample(logits, t=t, p=[p] * n, m=[0.01] * n, u=u, stride=vocab + 3)
    check_sample(logits, t=t, p=np.where(np.arange(n) % 2, 1.0, 0.43), k=np.where(np.arange(n) % 3, 0, vocab // 2 + 1), u=u)


@pytest.mark.parametrize("vocab", [30011, 151936])
def test_sample_shares_next_to_one(gpu, vocab):
    """Borders far down, where the rough sums say least."""
    rng = np.random.default_rng(vocab)
    p = 1 - np.array([3e-2, 1e-2, 1e-3, 3e-4, 1e-4, 4e-5, 1e-5, 1e-6, 2.0 ** -24])
    log(f"shares next to one of {vocab}")
    for t, dev_ in ((1.0, 2.0), (0.7, 1.5), (1.7, 1.0), (1.0, 0.1)):
        x = (rng.standard_normal((len(p), vocab)) * dev_).astype(F32)
        check_sample(x, t=[t] * len(p), p=p, u=1 - (rng.random(len(p)) * 0.02).astype(F32))
        check_sample(x, t=[t] * len(p), p=p, k=rng.integers(vocab // 50, vocab, len(p)), u=1 - (rng.random(len(p)) * 0.02).astype(F32))


def test_sample_tiny_temperatures(gpu):
    """Down to the type's smallest: the likeliest tokens share the draw."""
    rng = np.random.default_rng(14)
    for top in (0.0, -1.5, 3.0, 1e-39):
        x = (np.minimum(rng.standard_normal((6, 9000)) - 6, -0.5) + top).astype(F32)
        x[:, 4000], x[:, 7000] = top, top
        t = np.array([1e-30, 1e-37, 1e-38, 1e-40, 1e-45, 2.0 ** -100], F32)
        log(f"tiny temperatures below {top}")
        for u, token in ((0.3, 4000), (0.7, 7000)):
            for s in (dict(), dict(m=[0.5] * 6), dict(p=[0.9] * 6), dict(k=[4] * 6)):
                assert (check_sample(x, t=t, u=[u] * 6, **s) == token).all()


@pytest.mark.parametrize("top", [0.0, -0.0, 1e-39, 2.0 ** -85, -2.0 ** -85, 2.0 ** -100])
def test_sample_limits_at_tiny_temperatures(gpu, top):
    """Where 1 / t is infinite or next to it and the largest logit next to zero: k and p cut as ever, ties by rising
    index among them."""
    rng = np.random.default_rng(17)
    t = np.array([1e-30, 2.0 ** -100, 2.0 ** -101, 2.0 ** -120, 2.0 ** -126, 2.0 ** -130, 1e-40, 1e-42, 1e-45], F32)
    n, ties = len(t), [1234, 4000, 7000]
    x = (np.minimum(rng.standard_normal((n, 9000)) - 6, -0.5) + top).astype(F32)
    x[:, ties] = top
    log(f"limits at tiny temperatures below {top}")
    for s, kept in ((dict(k=[1] * n), 1), (dict(k=[2] * n), 2), (dict(p=[0.3] * n), 1), (dict(p=[0.6] * n), 2), (dict(p=[0.9] * n), 3),
                    (dict(k=[2] * n, p=[0.4] * n), 1), (dict(k=[2] * n, p=[0.6] * n), 2)):
        for u in (0.1, 0.6, 0.9):
            assert (check_sample(x, t=t, u=[u] * n, **s) == ties[int(u * kept)]).all()
    # logits a part of t apart, as far as there are such numbers next to `top`
    for part in (0.25, 1.0, 7.0):
        y = x.copy()
        y[:, 100:180] = (F32(top) - part * t[:, None].astype(np.float64) * np.arange(80)).astype(F32)
        for s in (dict(k=[3] * n), dict(p=[0.83] * n), dict(k=[17] * n, p=[0.771] * n), dict(p=[0.913] * n, m=[0.11] * n)):
            check_sample(y, t=t, u=rng.random(n), **s)


def test_half_of_two_ties_at_tiny_temperatures(gpu):
    """p of 0.5 of two equal weights is reached by the first."""
    t = np.array([1e-37, 2.0 ** -130, 1e-40, 1e-45], F32)
    x = np.full((4, 9000), -3.0, F32)
    x[:, 4000] = x[:, 7000] = 0.0
    log("half of two ties")
    assert (run_sample(x, t=t, p=[0.5] * 4, u=[0.7] * 4)[0] == 4000).all()


@pytest.mark.parametrize("top", [0.0, -0.0, 1e-39, 2.0 ** -85, -2.0 ** -85, 2.0 ** -100])
def test_sample_limits_at_tiny_temperatures(gpu, top):
    """Where 1 / t is infinite or next to it and the largest logit next to zero: k and p cut as ever, ties by rising
    index among them."""
    rng = np.random.default_rng(17)
    t = np.array([1e-30, 2.0 ** -100, 2.0 ** -101, 2.0 ** -120, 2.0 ** -126, 2.0 ** -130, 1e-40, 1e-42, 1e-45], F32)
    n, ties = len(t), [1234, 4000, 7000]
    x = (np.minimum(rng.standard_normal((n, 9000)) - 6, -0.5) + top).astype(F32)
    x[:, ties] = top
    log(f"limits at tiny temperatures below {top}")
    for s, kept in ((dict(k=[1] * n), 1), (dict(k=[2] * n), 2), (dict(p=[0.3] * n), 1), (dict(p=[0.6] * n), 2), (dict(p=[0.9] * n), 3),
                    (dict(k=[2] * n, p=[0.4] * n), 1), (dict(k=[2] * n, p=[0.6] * n), 2)):
        for u in (0.1, 0.6, 0.9):
            assert (check_sample(x, t=t, u=[u] * n, **s) == ties[int(u * kept)]).all()
    # logits a part of t apart, as far as there are such numbers next to `top`
    for part in (0.25, 1.0, 7.0):
        y = x.copy()
        y[:, 100:180] = (F32(top) - part * t[:, None].astype(np.float64) * np.arange(80)).astype(F32)
        for s in (dict(k=[3] * n), dict(p=[0.83] * n), dict(k=[17] * n, p=[0.771] * n), dict(p=[0.913] * n, m=[0.11] * n)):
            check_sample(y, t=t, u=rng.random(n), **s)


def test_half_of_two_ties_at_tiny_temperatures(gpu):
    """p of 0.5 of two equal weights is reached by the first."""
    t = np.array([1e-37, 2.0 ** -130, 1e-40, 1e-45], F32)
    x = np.full((4, 9000), -3.0, F32)
    x[:, 4000] = x[:, 7000] = 0.0
    log("half of two ties")
    assert (run_sample(x, t=t, p=[0.5] * 4, u=[0.7] * 4)[0] == 4000).all()


def test_sample_of_a_long_row(gpu):
    rng = np.random.default_rng(9)
    vocab = 2 ** 22 - 3
    log(f"row of {vocab}")
    x = rng.standard_normal((1, vocab), dtype=F32) * 3
    check_sample(x, k=[100], u=[0.3])
    check_sample(x, p=[0.9], u=[0.71])
    check_sample(x, u=[0.999])


def test_sample_misaligned_rows(gpu):
    """Rows that begin at any float."""
    import torch
    rng = np.random.default_rng(10)
    rows, vocab, stride = 5, 9001, 9003
    buf = rng.standard_normal(rows * stride + 4).astype(F32)
    d, s = native.SampleDesc(rows=rows, vocab=vocab, stride=stride), settings(rng, rows)
    n = native.sample_workspace_size(d)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    t = dev(buf)
    arrays = [dev(s[x]) for x in "tkpmu"]
    for off in range(4):
        token, lp = dev(np.zeros(rows, I32)), dev(np.zeros(rows, F32))
        log(f"offset {off}")
        native.sample(d, t.data_ptr() + 4 * off, *map(ptr, arrays), ptr(token), ptr(lp), ptr(ws), n, stream())
        for r in range(rows):
            row = buf[off + r * stride:off + r * stride + vocab]
            assert token.cpu().numpy()[r] == ref.sample(row, *(s[x][r] for x in "tkpmu"))[0]


def test_sample_without_log_probabilities(gpu):
    rng = np.random.default_rng(11)
    x, s = rng.standard_normal((6, 5000)).astype(F32), settings(rng, 6)
    log("no log-probabilities")
    with_lp = run_sample(x, **s)[0]
    assert np.array_equal(run_sample(x, **s, logprobs=False)[0], with_lp)


def test_sample_follows_the_distribution(gpu):
    """Even random numbers draw each token as often as its share: exactly, by counting."""
    rng = np.random.default_rng(12)
    row = (rng.standard_normal(50) * 1.5).astype(F32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(F32)
    log("shares")
    token = run_sample(np.tile(row, (n, 1)), t=np.full(n, 0.8), p=np.full(n, 0.9), u=u)[0]
    w, order = ref.weights(row, np.float64(F32(0.8)))
    keep = order[:int(np.searchsorted(np.cumsum(w[order]), float(F32(0.9)) * w.sum())) + 1]
    share = np.zeros(50)
    share[keep] = w[keep] / w[keep].sum()
    assert np.abs(np.bincount(token, minlength=50) - share * n).max() <= 1.0


def test_sample_rows_in_batches(gpu):
    """More rows than the workspace holds at a time, each with settings of its own."""
    rng = np.random.default_rng(15)
    rows, vocab = 2900, 301
    one = native.sample_workspace_size(native.SampleDesc(rows=1, vocab=vocab))
    assert native.sample_workspace_size(native.SampleDesc(rows=rows, vocab=vocab)) < rows * one   # batches
    log(f"batches of {rows}")
    s = settings(rng, rows)
    s["u"] = (np.floor(s["u"] * 1000) + F32(0.37)) / F32(1000)
    check_sample((rng.standard_normal((rows, vocab)) * 2).astype(F32), **s)


def test_two_samples_at_once(gpu):
    """On two streams, of different vocabularies, each with a workspace of its own; as one after the other."""
    import torch
    rng = np.random.default_rng(16)
    calls = []
    for rows, vocab in ((40, 150001), (64, 30000)):
        s = settings(rng, rows)
        d = native.SampleDesc(rows=rows, vocab=vocab)
        n = native.sample_workspace_size(d)
        bufs = [dev((rng.standard_normal((rows, vocab)) * 2).astype(F32)), *(dev(s[x]) for x in "tkpmu")]
        calls.append((d, bufs, torch.empty(n, dtype=torch.uint8, device="cuda"), n, torch.cuda.Stream()))
    results = []
    for together in (False, True):
        outs = [[(dev(np.zeros(c[0].rows, I32)), dev(np.zeros(c[0].rows, F32))) for _ in range(6)] for c in calls]
        torch.cuda.synchronize()
        log(f"together {together}")
        for i in range(6):
            for (d, bufs, ws, n, st), out in zip(calls, outs):
                native.sample(d, *map(ptr, bufs), *map(ptr, out[i]), ptr(ws), n, st.cuda_stream)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append([[t.cpu().numpy() for t in pair] for out in outs for pair in out])
    for a, b in zip(*results):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_sample_replayed_from_a_graph(gpu):
    """Captured once, replayed with other logits and settings; every replay as an eager call."""
    import torch
    rng = np.random.default_rng(13)
    rows, vocab = 11, 20011
    d = native.SampleDesc(rows=rows, vocab=vocab)
    n = native.sample_workspace_size(d)
    ws, ws2 = (torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for _ in range(2))
    x = dev(np.zeros((rows, vocab), F32))
    arrays = [dev(np.zeros(rows, I32 if c == "k" else F32)) for c in "tkpmu"]
    out, lp, out2, lp2 = (dev(np.zeros(rows, ty)) for ty in (I32, F32, I32, F32))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        native.sample(d, ptr(x), *map(ptr, arrays), ptr(out), ptr(lp), ptr(ws), n, side.cuda_stream)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            native.sample(d, ptr(x), *map(ptr, arrays), ptr(out), ptr(lp), ptr(ws), n, side.cuda_stream)
    for i in range(5):
        logits, s = (rng.standard_normal((rows, vocab)) * 2).astype(F32), settings(rng, rows)
        x.copy_(dev(logits))
        for c, a in zip("tkpmu", arrays):
            a.copy_(dev(s[c]))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        native.sample(d, ptr(x), *map(ptr, arrays), ptr(out2), ptr(lp2), ptr(ws2), n, stream())
        torch.cuda.synchronize()
        log(f"replay {i}")
        assert torch.equal(out, out2) and torch.equal(lp, lp2)
        assert [ref.sample(logits[r], *(s[c][r] for c in "tkpmu"))[0] for r in range(rows)] == out.tolist()
