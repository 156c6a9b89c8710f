"""What a server's loop needs around a step's attention, as cases that can be timed and checked.

A case is a dict of plain values. `kind` says which operator it is:

  plan     page tables, cumulative lengths, positions and slot maps of a step, built from the
           lengths that the requests want and a free list of pages, all on the device
           (native.paged_plan); with `commit` the step's end too: lengths advance, the pages of
           requests that ended go back to the free list (native.paged_commit)
  shared   attention of each request's new tokens over a paged cache where groups of requests
           share a prefix, which is read once for all of them (native.paged_shared_attention)
  sample   the next token of each row of logits by temperature, top-k, top-p and min-p from given
           random numbers, with its log-probability (native.sample)

With `own` false a pass computes the operator in elementary torch operations; with `own` true it
calls the framework. Activations and logits are fp32, caches fp32 or fp16.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

POSITIONS = 2 ** 31 - 4096   # positions from here on have no page


def _plan(name, requests, want, past, page, mix="tokens", commit=False, tight=False):
    case = {"kind": "plan", "requests": requests, "want": want, "past": past, "page": page, "mix": mix,
            "commit": commit, "tight": tight}
    return {"name": name, **case} if name else case


def _shared(name, groups, requests, prefix, kept, new, heads, kv_heads, dim, page, cache="f16"):
    case = {"kind": "shared", "groups": groups, "requests": requests, "prefix": prefix, "kept": kept, "new": new,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache}
    return {"name": name, **case} if name else case


def _sample(name, rows, vocab, how):
    case = {"kind": "sample", "rows": rows, "vocab": vocab, "how": how}
    return {"name": name, **case} if name else case


def listed():
    return [
        # 32 chats decoded together: a token each, a new page now and then
        _plan("plan_tokens", 32, 1, 4000, 16),
        # continuous batching: every sixteenth of 256 requests a chunk of a prompt, the others a token; the pool
        # holds pages for most of them, the rest wait
        _plan("plan_mixed", 256, 700, 3000, 16, mix="some", tight=True),
        # prompts that are scored and leave: pages taken and returned within one step
        _plan("plan_prompts", 64, 900, 0, 32, mix="ragged", commit=True),
        # four chats of a 0.5B-class model behind one system prompt
        _shared("shared_one", 1, 4, 700, 60, 1, 14, 2, 64, 16),
        # 32 chats of a 7B-class model behind a prompt of 4000 tokens
        _shared("shared_tokens", 1, 32, 4000, 300, 1, 28, 4, 128, 16),
        # 64 answers sampled over one long document
        _shared("shared_long", 1, 64, 16000, 500, 1, 28, 4, 128, 64),
        # two tenants' prompts, fp32 cache, pages that end inside any tile
        _shared("shared_groups_f32", 2, 16, 2000, 150, 1, 32, 8, 96, 24, cache="f32"),
        # eight questions of 64 tokens over one document
        _shared("shared_chunks", 1, 8, 6000, 0, 64, 28, 4, 128, 16),
        # one chat: top-k, top-p and min-p together
        _sample("sample_one", 1, 151936, "all"),
        # 64 chats, each with settings of its own
        _sample("sample_rows", 64, 151936, "mixed"),
        # 32 rows of a small vocabulary by temperature alone
        _sample("sample_temperature", 32, 32000, "temperature"),
        # 200 answers sampled at top-p
        _sample("sample_top_p", 200, 50001, "top_p"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan"] * 2 + ["shared"] * 4 + ["sample"] * 4)
    page = rng.choice([16, 16, 32, 64, 128, 8, 24, 10])
    if kind == "plan":
        mix = rng.choice(["tokens", "some", "ragged"])
        past = rng.choice([0, _log(rng, 1, 8000)])
        requests = _log(rng, 1, 256)
        want = 1 if mix == "tokens" else _log(rng, 2, 1000)
        while requests * want > 64 * 900 or requests * (past + want) > 64 * 16500:
            requests = max(1, requests * 3 // 4)
        # (a request that ends holds fresh tokens alone here, so that every pass meets the same lengths)
        return _plan(None, requests, want, past, page, mix, past == 0 and rng.random() < 0.7, rng.random() < 0.3)
    if kind == "shared":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 7, 8])
        dim = rng.choice([64, 128, 128, 128, 96, 80, 256])
        cache = rng.choice(["f16", "f16", "f32"])
        new = rng.choice([1, 1, 1, _log(rng, 2, 200)])
        groups = rng.choice([1, 1, 1, rng.randint(2, 4)])
        requests = groups * _log(rng, 2, 64 // groups if new == 1 else 8)
        prefix, kept = _log(rng, 100, 16000), rng.choice([0, _log(rng, 1, 1000)])
        while True:   # within the listed cases' cost
            c = _shared(None, groups, requests, prefix, kept, new, heads, kv, dim, page, cache)
            if work(c)["bytes"] <= 60e6 and work(c)["flops"] <= (4e9 if cache == "f32" else 14e9):
                return c
            requests = max(groups, requests * 3 // 4 // groups * groups)
            prefix, kept, new = prefix * 3 // 4, kept * 3 // 4, max(1, new * 3 // 4)
    vocab = _log(rng, 1000, 160000)
    rows = min(_log(rng, 1, 256), max(1, 64 * 151936 // vocab))
    return _sample(None, rows, vocab, rng.choice(["all", "mixed", "mixed", "temperature", "top_k", "top_p", "min_p"]))


# ---- inputs --------------------------------------------------------------------------------------

def _spread(i, salt):
    """A fixed number in [0, 1) for request i: lengths follow from the case alone."""
    return ((i + 1) * 0.6180339887498949 + salt * 0.3819) % 1.0


def _lengths(case):
    """(tokens wanted, tokens cached) of each request."""
    R = case["requests"]
    if case["kind"] == "plan":
        want, past = case["want"], case["past"]
        pasts = [int(round(past * _spread(i, 0))) for i in range(R)]
        if case["mix"] == "some":
            wants = [want if i % 16 == 5 else 1 for i in range(R)]
        elif case["mix"] == "ragged":
            wants = [max(1, int(round(want * (0.2 + 0.8 * _spread(i, 1))))) for i in range(R)]
        else:
            wants = [want] * R
        return wants, pasts
    own_past = [int(round(case["kept"] * (0.25 + 0.75 * _spread(i, 0)))) for i in range(R)]
    new = [case["new"] if i % 3 else max(1, case["new"] - 1) for i in range(R)]
    return new, [p + s for p, s in zip(own_past, _prefixes(case, per_request=True))]


def _prefixes(case, per_request=False):
    """The shared tokens of each group (or of each request's group): whole pages."""
    page, n = case["page"], case["groups"]
    shared = [max(1, int(case["prefix"] * (1 - 0.15 * g)) // page) * page for g in range(n)]
    return [shared[i * n // case["requests"]] for i in range(case["requests"])] if per_request else shared


def _ceil(a, b):
    return -(-a // b)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _plan_inputs(case, gen):
    wants, pasts = _lengths(case)
    R, ps = case["requests"], case["page"]
    # room for rows: all of what is wanted, or most of it
    tokens = sum(wants) if not case["tight"] else max(1, sum(wants) * 7 // 8)
    have = [_ceil(p, ps) for p in pasts]
    need = [_ceil(p + w, ps) - h for p, w, h in zip(pasts, wants, have)]
    free = sum(need) + 7 if not case["tight"] else max(1, sum(need) * 3 // 4)
    num_pages = sum(have) + free
    width = max(h + n for h, n in zip(have, need))
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)
    column = torch.arange(width, device="cuda")
    h = torch.tensor(have, device="cuda")
    at = (torch.cumsum(h, 0) - h)[:, None] + column
    table = torch.where(column < h[:, None], order[at.clamp(max=num_pages - 1)], -1).to(torch.int32)
    stack = torch.full((num_pages,), -1, dtype=torch.int32, device="cuda")
    stack[:free] = order[sum(have):]
    s = {"tokens": tokens, "num_pages": num_pages, "want": _int(wants), "past": _int(pasts), "table": table,
         "free": stack, "free_count": _int([free])}
    if case["commit"]:   # every request ends with the step
        s["done"] = torch.ones(R, dtype=torch.int32, device="cuda")
    return s


def _shared_inputs(case, gen):
    news, pasts = _lengths(case)
    R, ps, n = case["requests"], case["page"], case["groups"]
    prefixes, mine = _prefixes(case), _prefixes(case, per_request=True)
    bounds = [next(i for i in range(R + 1) if i == R or i * n // R >= g) for g in range(n + 1)]
    pages = [_ceil(p + w, ps) for p, w in zip(pasts, news)]
    num_pages = sum(prefixes) // ps + sum(p - m // ps for p, m in zip(pages, mine)) + 3
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32).cpu()
    table = torch.zeros(R, max(pages), dtype=torch.int32)
    at = 0
    for g in range(n):
        shared = order[at:at + prefixes[g] // ps]
        at += len(shared)
        for r in range(bounds[g], bounds[g + 1]):
            table[r, :len(shared)] = shared
            table[r, len(shared):pages[r]] = order[at:at + pages[r] - len(shared)]
            at += pages[r] - len(shared)
    cu = [0]
    for w in news:
        cu.append(cu[-1] + w)
    shape, dt = (num_pages, ps, case["kv_heads"], case["dim"]), torch.float16 if case["cache"] == "f16" else torch.float32
    normal = lambda *size: torch.randn(*size, device="cuda", generator=gen)   # noqa: E731
    return {"cu": _int(cu), "past": _int(pasts), "table": table.cuda(), "groups": _int(bounds), "shared": _int(prefixes),
            "k_cache": normal(*shape).to(dt), "v_cache": normal(*shape).to(dt), "tokens": cu[-1],
            "q": normal(cu[-1], case["heads"] * case["dim"]) * 1.5, "bounds": bounds, "prefixes": prefixes,
            "news": news, "pasts": pasts}


def _sample_inputs(case, gen):
    rows, vocab, how = case["rows"], case["vocab"], case["how"]
    rand = lambda: torch.rand(rows, device="cuda", generator=gen)   # noqa: E731
    # a language model's row: a broad bulk, and a few dozen likely tokens above it
    logits = torch.randn(rows, vocab, device="cuda", generator=gen) * 2 - 3
    likely = torch.arange(40, device="cuda") * (vocab // 40) + torch.randint(0, vocab // 40, (rows, 40), device="cuda", generator=gen)
    logits.scatter_(1, likely, 4 + 7 * torch.rand(rows, 40, device="cuda", generator=gen))
    s = {"logits": logits, "random": rand(), "temperature": 0.6 + 0.8 * rand(), "top_k": None, "top_p": None, "min_p": None}
    if how in ("all", "top_k", "mixed"):
        s["top_k"] = torch.randint(5, 200, (rows,), device="cuda", generator=gen).to(torch.int32)
    if how in ("all", "top_p", "mixed"):
        s["top_p"] = 0.8 + 0.19 * rand()
    if how in ("all", "min_p", "mixed"):
        s["min_p"] = 0.01 + 0.09 * rand()
    if how == "mixed":   # each row its own settings; every eighth the likeliest token
        i = torch.arange(rows, device="cuda")
        s["top_k"] = torch.where(i % 3 == 0, s["top_k"], 0).to(torch.int32)
        s["top_p"] = torch.where(i % 2 == 0, s["top_p"], 1.0)
        s["min_p"] = torch.where(i % 5 == 0, s["min_p"], 0.0)
        s["temperature"] = torch.where(i % 8 == 7, 0.0, s["temperature"])
    return s


def _inputs(case, seed):
    return {"plan": _plan_inputs, "shared": _shared_inputs, "sample": _sample_inputs}[case["kind"]](case, _generator(seed))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    ints = lambda *n: torch.empty(*n, dtype=torch.int32, device="cuda")   # noqa: E731
    if kind == "plan":
        s.update(cu=ints(case["requests"] + 1), used=ints(1), request=ints(s["tokens"]), position=ints(s["tokens"]),
                 slot=ints(s["tokens"]))
    if own:
        from modelsharp_amd import native
        if kind == "plan":
            s["desc"] = native.StepDesc(tokens=s["tokens"], requests=case["requests"], page_size=case["page"],
                                        num_pages=s["num_pages"], max_pages=s["table"].shape[1])
        elif kind == "shared":
            s["desc"] = native.PagedDesc(
                tokens=s["tokens"], requests=case["requests"], max_new=max(s["news"]),
                max_total=max(a + b for a, b in zip(s["news"], s["pasts"])), num_heads=case["heads"],
                kv_num_heads=case["kv_heads"], head_dim=case["dim"], page_size=case["page"],
                num_pages=s["k_cache"].shape[0], max_pages=s["table"].shape[1],
                cache_type=native.MS_HIP_DTYPE_F16 if case["cache"] == "f16" else native.MS_HIP_DTYPE_F32,
                local_window_size=-1, scale=0.0)
            mine = _prefixes(case, per_request=True)
            s["groups_desc"] = native.SharedDesc(
                groups=case["groups"], max_shared=max(s["prefixes"]),
                max_rest=max(a + b - c for a, b, c in zip(s["news"], s["pasts"], mine)))
            n = native.paged_shared_attention_workspace_size(s["desc"], s["groups_desc"])
            s["ws_bytes"], s["ws"] = n, torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
            s["out"] = torch.empty_like(s["q"])
        else:
            s["desc"] = native.SampleDesc(rows=case["rows"], vocab=case["vocab"])
            n = native.sample_workspace_size(s["desc"])
            s["ws_bytes"], s["ws"] = n, torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
            s["token"], s["logprob"] = ints(case["rows"]), torch.empty(case["rows"], device="cuda")
    torch.cuda.synchronize()
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    if own:
        return _framework(s)
    return {"plan": _plan_plain, "shared": _shared_plain, "sample": _sample_plain}[s["case"]["kind"]](s)


def _plan_outputs(s):
    names = ["cu", "used", "request", "position", "slot", "table"]
    if s["case"]["commit"]:
        names += ["past", "free", "free_count"]
    return {n: s[n] for n in names}


def _framework(s):
    from modelsharp_amd import native
    kind = s["case"]["kind"]
    st = torch.cuda.current_stream().cuda_stream
    opt = lambda t: None if t is None else t.data_ptr()   # noqa: E731
    if kind == "plan":
        native.paged_plan(s["desc"], s["want"].data_ptr(), s["past"].data_ptr(), s["free"].data_ptr(),
                          s["free_count"].data_ptr(), s["table"].data_ptr(), s["cu"].data_ptr(), s["used"].data_ptr(),
                          s["request"].data_ptr(), s["position"].data_ptr(), s["slot"].data_ptr(), st)
        if s["case"]["commit"]:
            native.paged_commit(s["desc"], s["cu"].data_ptr(), s["used"].data_ptr(), s["done"].data_ptr(), None,
                                s["past"].data_ptr(), s["table"].data_ptr(), s["free"].data_ptr(),
                                s["free_count"].data_ptr(), st)
        return _plan_outputs(s)
    if kind == "shared":
        native.paged_shared_attention(s["desc"], s["groups_desc"], s["q"].data_ptr(), s["cu"].data_ptr(),
                                      s["past"].data_ptr(), s["table"].data_ptr(), s["groups"].data_ptr(),
                                      s["shared"].data_ptr(), s["k_cache"].data_ptr(), s["v_cache"].data_ptr(),
                                      s["out"].data_ptr(), s["ws"].data_ptr(), s["ws_bytes"], st)
        return s["out"]
    native.sample(s["desc"], s["logits"].data_ptr(), opt(s["temperature"]), opt(s["top_k"]), opt(s["top_p"]),
                  opt(s["min_p"]), s["random"].data_ptr(), s["token"].data_ptr(), s["logprob"].data_ptr(),
                  s["ws"].data_ptr(), s["ws_bytes"], st)
    return {"token": s["token"], "logprob": s["logprob"]}


def _plan_plain(s):
    ps, T, NP = s["case"]["page"], s["tokens"], s["num_pages"]
    table, R, W = s["table"], s["table"].shape[0], s["table"].shape[1]
    want, past = s["want"].long().clamp(min=0), s["past"].long().clamp(min=0)
    have, pages = (past + ps - 1) // ps, (past + want + ps - 1) // ps
    fits = (want > 0) & (pages <= W) & (past + want <= POSITIONS)
    ask, need = want * fits, (pages - have) * fits
    count = s["free_count"].long().clamp(0, NP)
    served = fits & (torch.cumsum(ask, 0) <= T) & ((need == 0) | (torch.cumsum(need, 0) <= count))
    new, take = ask * served, need * served
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(new, 0)])
    base = torch.cumsum(take, 0) - take
    s["cu"].copy_(cu)
    s["used"].copy_(take.sum(0, keepdim=True))
    # page j of the step comes from the top of the stack
    column = torch.arange(W, device="cuda")
    j = base[:, None] + column - have[:, None]
    fresh = (column >= have[:, None]) & (column < (have + take)[:, None])
    table.copy_(torch.where(fresh, s["free"][(count - 1 - j).clamp(0, NP - 1)], table))
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    there, r = r < R, r.clamp(max=R - 1)
    pos = past[r] + t - cu[r]
    entry = table[r, (pos // ps).clamp(max=W - 1)].long()
    slot = torch.where((entry >= 0) & (entry < NP), entry * ps + pos % ps, -1)
    for name, x in (("request", r), ("position", pos), ("slot", slot)):
        s[name].copy_(torch.where(there, x, -1))
    if s["case"]["commit"]:
        done = s["done"] != 0
        after = past + new
        gone = done[:, None] & (column < ((after + ps - 1) // ps)[:, None])
        back = gone & (table >= 0) & (table < NP)
        place = (count - take.sum()) + torch.cumsum(back.reshape(-1).long(), 0) - 1
        place = torch.where(back.reshape(-1) & (place < NP), place, NP)
        stack = torch.cat([s["free"], s["free"].new_zeros(1)]).scatter(0, place, table.reshape(-1))
        s["free"].copy_(stack[:NP])
        s["free_count"].copy_((count - take.sum() + back.sum()).clamp(max=NP))
        table.copy_(torch.where(gone, -1, table))
        s["past"].copy_(torch.where(done, 0, after))
    return _plan_outputs(s)


def _shared_plain(s):
    c = s["case"]
    H, G, D, R, ps = c["heads"], c["kv_heads"], c["dim"], c["requests"], c["page"]
    scale = 1.0 / math.sqrt(D)
    t = torch.arange(s["tokens"], device="cuda")
    r = torch.bucketize(t, s["cu"][1:].long(), right=True)
    i = t - s["cu"].long()[r]
    q = s["q"].reshape(-1, G, H // G, D)
    out = torch.empty_like(q)
    M = max(s["news"])
    for g, P in enumerate(s["prefixes"]):
        first, last = s["bounds"][g], s["bounds"][g + 1]
        a, b = sum(s["news"][:first]), sum(s["news"][:last])
        rows = q[a:b].permute(1, 0, 2, 3)                                        # [G, tokens, H / G, D]
        # the prefix, once for every row of the group
        shared = s["table"][first, :P // ps].long()
        keys, values = (x[shared].float().reshape(P, G, D).permute(1, 0, 2) for x in (s["k_cache"], s["v_cache"]))
        near = torch.matmul(rows.reshape(G, -1, D), keys.transpose(1, 2).contiguous()) * scale
        near = near.reshape(G, b - a, H // G, P)
        # what follows it, each request's own
        width = max(p + w - P for p, w in zip(s["pasts"][first:last], s["news"][first:last]))
        at = P + torch.arange(width, device="cuda")
        table = s["table"][first:last].long()
        where = table[:, (at // ps).clamp(max=table.shape[1] - 1)] * ps + at % ps
        mine = lambda x: x.reshape(-1, G, D)[where].float().permute(0, 2, 1, 3)   # noqa: E731
        padded = torch.zeros(last - first, M, G, H // G, D, device="cuda")
        rr, ii = r[a:b] - first, i[a:b]
        padded[rr, ii] = q[a:b]
        padded = padded.permute(0, 2, 1, 3, 4).reshape(last - first, G, -1, D)
        far = torch.matmul(padded, mine(s["k_cache"]).transpose(2, 3).contiguous()) * scale
        far = far.reshape(last - first, G, M, H // G, width).permute(0, 2, 1, 3, 4)[rr, ii].permute(1, 0, 2, 3)
        pos = s["past"].long()[r[a:b]] + ii
        far = far.masked_fill((at > pos[:, None])[None, :, None], -math.inf)
        top = torch.maximum(near.amax(dim=-1, keepdim=True), far.amax(dim=-1, keepdim=True))
        near, far = torch.exp(near - top), torch.exp(far - top)
        total = near.sum(dim=-1, keepdim=True) + far.sum(dim=-1, keepdim=True)
        o = torch.matmul(near.reshape(G, -1, P), values).reshape(G, b - a, H // G, D)
        w = torch.zeros(last - first, M, G, H // G, width, device="cuda")
        w[rr, ii] = far.permute(1, 0, 2, 3)
        # the last page's rows past a request's end hold nothing of its
        ends = (s["past"] + s["cu"][1:] - s["cu"][:-1]).long()[first:last]
        own_values = mine(s["v_cache"]) * (at < ends[:, None])[:, None, :, None]
        w = w.permute(0, 2, 1, 3, 4).reshape(last - first, G, -1, width)
        o2 = torch.matmul(w, own_values).reshape(last - first, G, M, H // G, D).permute(0, 2, 1, 3, 4)[rr, ii]
        out[a:b] = ((o + o2.permute(1, 0, 2, 3)) / total).permute(1, 0, 2, 3)
    return out.reshape(s["tokens"], H * D)


def _sample_plain(s):
    logits, rows, V = s["logits"], s["case"]["rows"], s["case"]["vocab"]
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)   # ties: the lowest index first
    # sums and what lies next to a border in 64 bits
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((value.double() - value[:, :1].double()) / torch.where(greedy, 1.0, t))
    rank = torch.arange(V, device="cuda")
    keep = torch.where(greedy, rank == 0, rank >= 0)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((rank < k) | (k <= 0))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        kept = w * keep
        before = torch.cumsum(kept, dim=1) - kept
        keep = keep & ((before < p * kept.sum(dim=1, keepdim=True)) | (p >= 1))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter(1, order, w * keep)   # by index again
    total = kept.sum(dim=1, keepdim=True)
    reached = torch.cumsum(kept, dim=1) > s["random"].double()[:, None] * total
    token = reached.to(torch.int32).argmax(dim=1)            # the first
    chosen = kept.gather(1, token[:, None])
    return {"token": token.to(torch.int32), "logprob": torch.log(chosen / total)[:, 0].float()}


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind = case["kind"]
    wants, pasts = ([], []) if kind == "sample" else _lengths(case)
    if kind == "plan":
        ps, R, T = case["page"], case["requests"], sum(wants)
        fresh = sum(_ceil(p + w, ps) - _ceil(p, ps) for p, w in zip(pasts, wants))
        touched = sum(_ceil(p + w, ps) - p // ps for p, w in zip(pasts, wants))
        both = 2 * 4 * (R + 2 * fresh) if case["commit"] else 0   # lengths advance, entries leave the table for the stack
        return {"bytes": 4 * (3 * R + 1 + 3 * T + 2 * fresh + touched) + both, "flops": 4 * T}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    size = 2 if case["cache"] == "f16" else 4
    mine = _prefixes(case, per_request=True)
    keys = sum(_prefixes(case)) + sum(p + w - m for p, w, m in zip(pasts, wants, mine))
    pairs = sum(w * p + w * (w + 1) // 2 for p, w in zip(pasts, wants))
    return {"bytes": 8 * sum(wants) * H * D + 2 * keys * G * D * size, "flops": 4 * pairs * H * D}


# ---- the definition in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"plan": _plan64, "shared": _shared64, "sample": _sample64}[case["kind"]](case, s)


def _plan64(case, s):
    """One request after the other, on the host."""
    ps, R, T = case["page"], case["requests"], s["tokens"]
    want, past, free, table = (s[n].cpu().numpy().astype(np.int64) for n in ("want", "past", "free", "table"))
    count, W = int(s["free_count"].item()), table.shape[1]
    cu, out, used, asked, wanted = [0], [], 0, 0, 0
    for r in range(R):
        served = 0
        pages = _ceil(past[r] + want[r], ps)
        if want[r] > 0 and pages <= W and past[r] + want[r] <= POSITIONS:
            missing = pages - _ceil(past[r], ps)
            asked, wanted = asked + want[r], wanted + missing
            if asked <= T and (missing == 0 or wanted <= count):
                served = int(want[r])
                for col in range(_ceil(past[r], ps), pages):
                    table[r, col] = free[count - 1 - used]
                    used += 1
        for i in range(served):
            pos = past[r] + i
            out.append((r, pos, table[r, pos // ps] * ps + pos % ps))
        cu.append(cu[-1] + served)
    out += [(-1, -1, -1)] * (T - len(out))
    whole = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32)   # noqa: E731
    request, position, slot = zip(*out)
    result = {"cu": whole(cu), "used": whole([used]), "request": whole(request), "position": whole(position),
              "slot": whole(slot)}
    if case["commit"]:
        count -= used
        for r in range(R):
            for col in range(_ceil(past[r] + cu[r + 1] - cu[r], ps)):
                free[count] = table[r, col]
                table[r, col] = -1
                count += 1
    result["table"] = whole(table)
    if case["commit"]:
        result.update(past=whole([0] * R), free=whole(free), free_count=whole([count]))
    return result


def _shared64(case, s):
    H, G, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(s["tokens"], H, D, dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, p) in enumerate(zip(s["news"], s["pasts"])):
        key = torch.arange(p + n, device="cuda")
        row = s["table"][b, key // ps].long() * ps + key % ps
        k, v = (s[c].reshape(-1, G, D)[row].double() for c in ("k_cache", "v_cache"))
        hidden = key[None] > torch.arange(p, p + n, device="cuda")[:, None]
        for h in range(H):
            g = h // (H // G)
            x = s["q"][t:t + n, h * D:(h + 1) * D].double() @ k[:, g].t().contiguous() / math.sqrt(D)
            out[t:t + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v[:, g].contiguous()
        t += n
    return out.reshape(s["tokens"], -1)


def _sample64(case, s):
    """Row by row on the host: probabilities, cut from the likeliest on, then drawn by index."""
    logits = s["logits"].cpu().numpy().astype(np.float64)
    read = lambda n, off: np.full(case["rows"], off) if s[n] is None else s[n].cpu().numpy().astype(np.float64)   # noqa: E731
    temperature, k, p, m = read("temperature", 1.0), read("top_k", 0), read("top_p", 1.0), read("min_p", 0.0)
    random, tokens, logs = read("random", 0.0), [], []
    for r, row in enumerate(logits):
        if temperature[r] <= 0:
            tokens.append(int(np.argmax(row)))
            logs.append(0.0)
            continue
        x = row / temperature[r]
        prob = np.exp(x - x.max())
        order = np.lexsort((np.arange(len(row)), -row))
        n = min(int(k[r]), len(row)) if k[r] > 0 else len(row)
        sums = np.cumsum(prob[order[:n]])
        if p[r] < 1:
            n = min(n, int(np.searchsorted(sums, p[r] * sums[-1], side="left")) + 1)
        n = max(1, min(n, int((prob[order[:n]] >= m[r]).sum())))
        left = np.sort(order[:n])
        sums = np.cumsum(prob[left])
        at = min(int(np.searchsorted(sums, random[r] * sums[-1], side="right")), n - 1)
        tokens.append(int(left[at]))
        logs.append(math.log(prob[left[at]] / sums[-1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logs, dtype=torch.float64)}
