"""The operators of a serving step over many requests, as cases that can be timed and checked.

A case is a dict of plain values. `kind` says which operator it is:

  attend   attention of each request's new tokens over its keys and values in a paged cache
           (native.paged_attention): single tokens, chunks of a prompt, both in one batch
  append   norms of queries and keys per head, the position rotation, and the append of the new
           keys and values to the paged cache (native.paged_append)
  rotate   the same norms and rotation onto contiguous rows, for GroupQueryAttention
           (native.qk_norm_rotary)
  lora     low-rank adapters of many requests beside a shared projection (native.lora)

With `own` false a pass computes the operator in elementary torch operations in 32 bits; with
`own` true it calls the framework. Activations are fp32, as everywhere in the framework; caches
and adapters are fp32 or fp16.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6


def _attend(name, requests, new, past, heads, kv_heads, dim, page, cache="f16", window=-1, mix="even"):
    case = {"kind": "attend", "requests": requests, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "cache": cache, "window": window, "mix": mix}
    return {"name": name, **case} if name else case


def _append(name, requests, new, past, heads, kv_heads, dim, page, cache="f16", mix="even", rot=1.0, pairs="halves",
            norm=True):
    case = {"kind": "append", "requests": requests, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "cache": cache, "mix": mix, "rot": rot, "pairs": pairs, "norm": norm}
    return {"name": name, **case} if name else case


def _rotate(name, tokens, heads, kv_heads, dim, rot=1.0, pairs="halves", norm=True):
    case = {"kind": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "pairs": pairs, "norm": norm}
    return {"name": name, **case} if name else case


def _lora(name, tokens, K, N, adapters, rank, requests, weights="f16"):
    case = {"kind": "lora", "tokens": tokens, "K": K, "N": N, "adapters": adapters, "rank": rank,
            "requests": requests, "weights": weights}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one chat on a 0.5B-class model: one token over a few hundred cached ones
        _attend("attend_one", 1, 1, 700, 14, 2, 64, 16),
        # 32 chats on a 7B-class model decoded together, histories of 1000 to 4000 tokens
        _attend("attend_tokens", 32, 1, 4095, 28, 4, 128, 16),
        # eight long histories decoded together from an fp32 cache
        _attend("attend_tokens_f32", 8, 1, 8000, 32, 8, 128, 32, cache="f32"),
        # the next 512 tokens of a long document, 16000 tokens of it already cached
        _attend("attend_chunk_long", 1, 512, 16000, 28, 4, 128, 64),
        # five fresh prompts of odd lengths in one batch
        _attend("attend_prompts", 5, 700, 0, 28, 4, 128, 16, mix="ragged"),
        # two chunks under a sliding window, fp32 cache, pages that end inside any tile
        _attend("attend_window_f32", 2, 300, 1500, 32, 8, 96, 24, cache="f32", window=1024, mix="ragged"),
        # continuous batching: one chunk of a prompt beside fifteen chats
        _attend("attend_mixed", 16, 400, 3000, 28, 4, 128, 16, mix="one"),
        # the queries and keys of eight chats' next tokens
        _append("append_tokens", 8, 1, 2000, 28, 4, 128, 16),
        # four chunks of prompts
        _append("append_chunk", 4, 512, 1000, 28, 4, 128, 16),
        # an odd prompt on a 0.5B-class model before GroupQueryAttention
        _rotate("rotate_prompt", 1501, 14, 2, 64),
        # 32 chats with 16 adapters on a 7B-class projection, one token each
        _lora("lora_tokens", 32, 3584, 3584, 16, 16, 32),
        # four prompts, each with its own adapter, on a 7B-class MLP projection
        _lora("lora_prompt", 2048, 4096, 11008, 4, 64, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 7, 8]), kv


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["append"] * 2 + ["rotate"] + ["lora"] * 3)
    cache = rng.choice(["f16", "f16", "f32"])
    page = rng.choice([16, 16, 32, 64, 128, 256, 8, 24, 10])
    if kind == "attend":
        heads, kv = _heads(rng)
        dim = rng.choice([64, 128, 128, 128, 96, 80, 256])
        window = rng.choice([-1, -1, -1, _log(rng, 16, 4000)])
        mix = rng.choice(["tokens", "tokens", "chunk", "prompts", "one"])
        requests = 1 if mix == "chunk" and rng.random() < 0.5 else _log(rng, 1, 64 if mix == "tokens" else 16)
        new = 1 if mix == "tokens" else _log(rng, 2, 1024)
        past = 0 if mix == "prompts" else _log(rng, 1, 16000)
        while True:   # within the listed cases' cost
            c = _attend(None, requests, new, past, heads, kv, dim, page, cache, window,
                        "one" if mix == "one" else "ragged" if requests > 1 and new > 1 else "even")
            padded = 4.0 * requests * new * heads * dim * (past + new)
            if work(c)["bytes"] <= 300e6 and padded <= (30e9 if cache == "f32" else 100e9) and \
                    requests * (past + new) * kv * dim <= 2.5e8:
                return c
            requests, new, past = max(1, requests * 3 // 4), max(2 if new > 1 else 1, new * 3 // 4), past * 3 // 4
    rot, pairs = rng.choice([1.0, 1.0, 0.5]), rng.choice(["halves", "halves", "neighbours"])
    norm = rng.random() < 0.8
    if kind == "append":
        heads, kv = _heads(rng)
        dim = rng.choice([64, 128, 128, 96, 80, 256])
        new = rng.choice([1, 1, _log(rng, 2, 1024)])
        requests = _log(rng, 1, 64 if new == 1 else 8)
        while requests * new * (heads + 2 * kv) * dim > 2048 * 36 * 128:
            new = max(1, new * 3 // 4)
        return _append(None, requests, new, _log(rng, 1, 4000), heads, kv, dim, page, cache,
                       "ragged" if new > 1 and requests > 1 else "even", rot, pairs, norm)
    if kind == "rotate":
        heads, kv = _heads(rng)
        dim = rng.choice([64, 128, 96, 256])
        return _rotate(None, min(_log(rng, 1, 4096), 2048 * 4608 // ((heads + kv) * dim)), heads, kv, dim, rot, pairs,
                       norm)
    K, N = (max(64, _log(rng, 256, 11008) // 8 * 8) for _ in range(2))
    tokens = rng.choice([rng.randint(1, 64), _log(rng, 1, 2048)])
    tokens = max(1, min(tokens, 2048 * (4096 + 11008) // (K + N)))
    requests = max(1, min(tokens, _log(rng, 1, 64)))
    return _lora(None, tokens, K, N, _log(rng, 1, 32), rng.choice([4, 8, 16, 16, 32, 64, 20]), requests,
                 rng.choice(["f16", "f16", "f32"]))


# ---- inputs --------------------------------------------------------------------------------------

def _spread(i, salt):
    """A fixed number in [0, 1) for request i: lengths follow from the case alone."""
    return ((i + 1) * 0.6180339887498949 + salt * 0.3819) % 1.0


def _lengths(case):
    """(new tokens, cached tokens) of each request."""
    R, new, past = case["requests"], case["new"], case["past"]
    pasts = [past if R == 1 else int(round(past * (0.25 + 0.75 * _spread(i, 0)))) for i in range(R)]
    if case["mix"] == "one":
        news = [new if i == R // 2 else 1 for i in range(R)]
    elif case["mix"] == "ragged":
        news = [max(1, int(round(new * (0.3 + 0.7 * _spread(i, 1))))) for i in range(R)]
    else:
        news = [new] * R
    return news, pasts


def _pairs(case):
    """(query, key) pairs the mask leaves, and keys that some query sees, over all requests."""
    pairs = keys = 0
    w = case.get("window", -1)
    for n, p in zip(*_lengths(case)):
        if w < 0:
            pairs += n * p + n * (n + 1) // 2
            keys += p + n
        else:
            pairs += sum(min(w, p + i + 1) for i in range(n))
            keys += min(p + n, w + n - 1) if w else 0
    return pairs, keys


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _half_dims(case):
    return max(1, int(case["dim"] * case["rot"]) // 2)


def _tables(case, rows):
    half = _half_dims(case)
    ang = torch.outer(torch.arange(rows, dtype=torch.float64),
                      1.0 / 10000 ** (torch.arange(half, dtype=torch.float64) / half))
    return torch.cos(ang).float().cuda(), torch.sin(ang).float().cuda()


def _cache_type(case):
    return torch.float16 if case["cache"] == "f16" else torch.float32


def _paged(case, gen):
    """The batch's lengths and page table, and a cache whose pages lie in any order."""
    news, pasts = _lengths(case)
    R, ps = case["requests"], case["page"]
    pages = [-(-(n + p) // ps) for n, p in zip(news, pasts)]
    width = max(pages)
    num_pages = sum(pages) + 3
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(R, width, dtype=torch.int32)
    at = torch.arange(sum(pages), dtype=torch.int32)
    first = 0
    for r, n in enumerate(pages):
        table[r, :n] = at[first:first + n]
        first += n
    table = order[table.cuda().long()].contiguous()
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    shape = (num_pages, ps, case["kv_heads"], case["dim"])
    return {"cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
            "past": torch.tensor(pasts, dtype=torch.int32, device="cuda"), "table": table,
            "k_cache": _normal(gen, *shape).to(_cache_type(case)), "v_cache": _normal(gen, *shape).to(_cache_type(case)),
            "tokens": cu[-1], "max_new": max(news), "max_total": max(n + p for n, p in zip(news, pasts))}


def _inputs(case, seed):
    """The tensors of a case from the seed alone."""
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "attend":
        s = _paged(case, gen)
        s["q"] = _normal(gen, s["tokens"], case["heads"] * case["dim"]) * 1.5
        return s
    if kind in ("append", "rotate"):
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        if kind == "append":
            s = _paged(case, gen)
            # the projections' packed rows [q | k | v]
            s["qkv"] = _normal(gen, s["tokens"], (H + 2 * G) * D) * 2.0
            rows = s["max_total"]
        else:
            s = {"tokens": case["tokens"], "q": _normal(gen, case["tokens"], H * D) * 2.0,
                 "k": _normal(gen, case["tokens"], G * D) * 2.0}
            rows = 2 * case["tokens"] + 8
            s["positions"] = torch.arange(case["tokens"], dtype=torch.int32, device="cuda") + case["tokens"] // 3
        s["gq"] = torch.rand(D, device="cuda", generator=gen) + 0.5 if case["norm"] else None
        s["gk"] = torch.rand(D, device="cuda", generator=gen) + 0.5 if case["norm"] else None
        s["cos"], s["sin"] = _tables(case, rows)
        return s
    T, K, N, A, r, R = (case[k] for k in ("tokens", "K", "N", "adapters", "rank", "requests"))
    dt = torch.float16 if case["weights"] == "f16" else torch.float32
    s = {"x": _normal(gen, T, K), "base": _normal(gen, T, N), "a": (_normal(gen, A, r, K) / math.sqrt(K)).to(dt),
         "b": (_normal(gen, A, N, r) * 0.1).to(dt)}
    # adapters of 16 rows or more differ in rank: rows past an adapter's rank are not its own
    ranks = [r if r < 16 or i % 3 else r // 2 for i in range(A)]
    s["ranks"] = torch.tensor(ranks, dtype=torch.int32, device="cuda")
    s["scales"] = torch.rand(A, device="cuda", generator=gen) + 0.5
    # each request's tokens lie together; in a large batch every ninth request has no adapter
    which = torch.randint(0, A, (R,), device="cuda", generator=gen)
    if R >= 9:
        which[8::9] = -1
    s["adapters"] = which[(torch.arange(T, device="cuda") * R) // T].to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if own:
        from modelsharp_amd import native
        empty = lambda *n: torch.empty(*n, device="cuda")   # noqa: E731
        if kind in ("attend", "append"):
            H, G, D = case["heads"], case["kv_heads"], case["dim"]
            s["desc"] = native.PagedDesc(
                tokens=s["tokens"], requests=case["requests"], max_new=s["max_new"], max_total=s["max_total"],
                num_heads=H, kv_num_heads=G, head_dim=D, page_size=case["page"], num_pages=s["k_cache"].shape[0],
                max_pages=s["table"].shape[1],
                cache_type=native.MS_HIP_DTYPE_F16 if case["cache"] == "f16" else native.MS_HIP_DTYPE_F32,
                local_window_size=case.get("window", -1), scale=0.0)
        if kind == "attend":
            s["ws_bytes"] = native.paged_attention_workspace_size(s["desc"])
            s["ws"] = torch.empty(max(16, s["ws_bytes"]), dtype=torch.uint8, device="cuda")
            s["out"] = empty(s["tokens"], H * D)
        elif kind == "append":
            d = s["desc"]
            d.q_stride = d.k_stride = d.v_stride = (H + 2 * G) * D
            d.do_rotary, d.rotary_interleaved = 1, int(case["pairs"] == "neighbours")
            d.cos_rows, d.cos_cols = s["cos"].shape
            d.eps = EPS
            s["q_out"] = empty(s["tokens"], H * D)
        elif kind == "rotate":
            s["desc"] = native.QkNormDesc(
                tokens=s["tokens"], num_heads=case["heads"], kv_num_heads=case["kv_heads"], head_dim=case["dim"],
                do_rotary=1, rotary_interleaved=int(case["pairs"] == "neighbours"), cos_rows=s["cos"].shape[0],
                cos_cols=s["cos"].shape[1], eps=EPS)
            s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        else:
            s["desc"] = native.LoraDesc(
                tokens=case["tokens"], K=case["K"], N=case["N"], adapters=case["adapters"], max_rank=case["rank"],
                weight_type=native.MS_HIP_DTYPE_F16 if case["weights"] == "f16" else native.MS_HIP_DTYPE_F32)
            s["ws_bytes"] = native.lora_workspace_size(s["desc"])
            s["ws"] = torch.empty(max(16, s["ws_bytes"]), dtype=torch.uint8, device="cuda")
            s["y"] = torch.empty_like(s["base"])
    torch.cuda.synchronize()
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    if own:
        return _framework(s)
    return {"attend": _attend_plain, "append": _append_plain, "rotate": _rotate_plain,
            "lora": _lora_plain}[s["case"]["kind"]](s)


def _framework(s):
    from modelsharp_amd import native
    kind = s["case"]["kind"]
    st = torch.cuda.current_stream().cuda_stream
    if kind == "attend":
        native.paged_attention(s["desc"], s["q"].data_ptr(), s["cu"].data_ptr(), s["past"].data_ptr(),
                               s["table"].data_ptr(), s["k_cache"].data_ptr(), s["v_cache"].data_ptr(),
                               s["out"].data_ptr(), s["ws"].data_ptr(), s["ws_bytes"], st)
        return s["out"]
    opt = lambda t: None if t is None else t.data_ptr()   # noqa: E731
    if kind == "append":
        c, q = s["case"], s["qkv"].data_ptr()
        k = q + 4 * c["heads"] * c["dim"]
        native.paged_append(s["desc"], q, k, k + 4 * c["kv_heads"] * c["dim"], opt(s["gq"]), opt(s["gk"]),
                            s["cu"].data_ptr(), s["past"].data_ptr(), s["table"].data_ptr(), s["cos"].data_ptr(),
                            s["sin"].data_ptr(), s["q_out"].data_ptr(), s["k_cache"].data_ptr(),
                            s["v_cache"].data_ptr(), st)
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "rotate":
        native.qk_norm_rotary(s["desc"], s["q"].data_ptr(), s["k"].data_ptr(), opt(s["gq"]), opt(s["gk"]),
                              s["positions"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(),
                              s["q_out"].data_ptr(), s["k_out"].data_ptr(), st)
        return {"q": s["q_out"], "k": s["k_out"]}
    native.lora(s["desc"], s["x"].data_ptr(), s["a"].data_ptr(), s["b"].data_ptr(), s["ranks"].data_ptr(),
                s["scales"].data_ptr(), s["adapters"].data_ptr(), s["base"].data_ptr(), s["y"].data_ptr(),
                s["ws"].data_ptr(), s["ws_bytes"], st)
    return s["y"]


def _places(s):
    """(request, place among its new tokens, position) of every token."""
    t = torch.arange(s["tokens"], device="cuda")
    r = torch.bucketize(t, s["cu"][1:].long(), right=True)
    i = t - s["cu"].long()[r]
    return r, i, s["past"].long()[r] + i


def _attend_plain(s):
    c = s["case"]
    H, G, D, R = c["heads"], c["kv_heads"], c["dim"], c["requests"]
    r, i, _ = _places(s)
    q = torch.zeros(R, s["max_new"], H, D, device="cuda")
    q[r, i] = s["q"].reshape(-1, H, D)
    q = q.reshape(R, s["max_new"], G, H // G, D).permute(0, 2, 3, 1, 4).reshape(R, G, -1, D)
    table = s["table"].long()
    keys = s["k_cache"][table].float().reshape(R, -1, G, D).permute(0, 2, 3, 1).contiguous()
    values = s["v_cache"][table].float().reshape(R, -1, G, D).permute(0, 2, 1, 3).contiguous()
    pos = s["past"].long()[:, None] + torch.arange(s["max_new"], device="cuda")
    key = torch.arange(keys.shape[3], device="cuda")
    keep = key <= pos[:, :, None]
    if c["window"] >= 0:
        keep = keep & (key > pos[:, :, None] - c["window"])
    # the last page's rows past a request's end hold nothing of its
    values = values * (key < (s["past"].long() + s["cu"][1:] - s["cu"][:-1])[:, None])[:, None, :, None]
    score = torch.matmul(q, keys) * (1.0 / math.sqrt(D))
    score = score.reshape(R, G, H // G, s["max_new"], -1).masked_fill(~keep[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(dim=-1, keepdim=True)
    out = torch.matmul(w.reshape(R, G, -1, w.shape[-1]), values).reshape(R, G, H // G, s["max_new"], D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 3, 1, 2, 4)[r, i].reshape(-1, H * D)


def _normed_rotated(s, x, gamma, pos):
    """x [tokens, heads, D]: the norm of each head, then the rotation by its token's position."""
    c = s["case"]
    if gamma is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * gamma
    half = s["cos"].shape[1]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if c["pairs"] == "halves":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1)


def _append_plain(s):
    c = s["case"]
    H, G, D, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    r, _, pos = _places(s)
    q, k, v = s["qkv"].split([H * D, G * D, G * D], dim=1)
    q = _normed_rotated(s, q.reshape(-1, H, D), s["gq"], pos)
    k = _normed_rotated(s, k.reshape(-1, G, D), s["gk"], pos)
    page, slot = s["table"].long()[r, pos // ps], pos % ps
    s["k_cache"][page, slot] = k.to(s["k_cache"].dtype)
    s["v_cache"][page, slot] = v.reshape(-1, G, D).to(s["v_cache"].dtype)
    return {"q": q.reshape(-1, H * D), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rotate_plain(s):
    c = s["case"]
    pos = s["positions"].long()
    return {n: _normed_rotated(s, s[n].reshape(c["tokens"], -1, c["dim"]), s["g" + n], pos).reshape(c["tokens"], -1)
            for n in ("q", "k")}


def _lora_plain(s):
    c = s["case"]
    T, K, N, A, rank = (c[k] for k in ("tokens", "K", "N", "adapters", "rank"))
    h = torch.matmul(s["x"], s["a"].float().reshape(A * rank, K).t()).reshape(T, A, rank)
    mine = s["adapters"].long()[:, None] == torch.arange(A, device="cuda")
    row = torch.arange(rank, device="cuda") < s["ranks"][:, None]
    h = h * (mine[:, :, None] & row) * s["scales"][:, None]
    b = s["b"].float().permute(0, 2, 1).reshape(A * rank, N)
    return s["base"] + torch.matmul(h.reshape(T, A * rank), b)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "lora":
        T, K, N, A, r, R = (case[k] for k in ("tokens", "K", "N", "adapters", "rank", "requests"))
        size = 2 if case["weights"] == "f16" else 4
        return {"bytes": 4 * T * (K + 2 * N) + min(A, R) * r * (K + N) * size, "flops": 2 * T * r * (K + N)}
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "rotate":
        T = case["tokens"]
        return {"bytes": 4 * T * (2 * (H + G) * D + 2 * _half_dims(case)), "flops": 8 * T * (H + G) * D}
    size = 2 if case["cache"] == "f16" else 4
    T = sum(_lengths(case)[0])
    if kind == "append":
        return {"bytes": 4 * T * ((2 * H + 2 * G) * D + 2 * _half_dims(case)) + size * T * 2 * G * D,
                "flops": 8 * T * (H + G) * D}
    pairs, keys = _pairs(case)
    return {"bytes": 8 * T * H * D + 2 * keys * G * D * size, "flops": 4 * pairs * H * D}


# ---- the definition in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "lora":
        y = s["base"].double()
        for a in range(case["adapters"]):
            t = torch.nonzero(s["adapters"] == a)[:, 0]
            r = int(s["ranks"][a])
            low = s["x"][t].double() @ s["a"][a, :r].double().t().contiguous()
            y[t] += float(s["scales"][a].double()) * (low @ s["b"][a, :, :r].double().t().contiguous())
        return y
    G, D = case["kv_heads"], case["dim"]
    if kind == "rotate":
        return {n: _heads64(case, s, s[n].double().reshape(case["tokens"], -1, D), s["g" + n],
                            s["positions"].long()).reshape(case["tokens"], -1) for n in ("q", "k")}
    news, pasts = _lengths(case)
    H, ps = case["heads"], case["page"]
    if kind == "append":
        qkv = s["qkv"].double().reshape(s["tokens"], H + 2 * G, D)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        out = torch.empty(s["tokens"], H, D, dtype=torch.float64, device="cuda")
        t = 0
        for b, (n, p) in enumerate(zip(news, pasts)):
            pos = torch.arange(p, p + n, device="cuda")
            out[t:t + n] = _heads64(case, s, qkv[t:t + n, :H], s["gq"], pos)
            row = s["table"][b, pos // ps].long() * ps + pos % ps
            kc.view(-1, G, D)[row] = _heads64(case, s, qkv[t:t + n, H:H + G], s["gk"], pos)
            vc.view(-1, G, D)[row] = qkv[t:t + n, H + G:]
            t += n
        return {"q": out.reshape(s["tokens"], -1), "k_cache": kc, "v_cache": vc}
    out = torch.empty(s["tokens"], H, D, dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        key = torch.arange(p + n, device="cuda")
        row = s["table"][b, key // ps].long() * ps + key % ps
        k, v = (s[c].reshape(-1, G, D)[row].double() for c in ("k_cache", "v_cache"))
        at = torch.arange(p, p + n, device="cuda")[:, None]
        keep = key[None] <= at
        if case["window"] >= 0:
            keep &= key[None] > at - case["window"]
        for h in range(H):
            g = h // (H // G)
            x = s["q"][t:t + n, h * D:(h + 1) * D].double() @ k[:, g].t().contiguous() / math.sqrt(D)
            w = torch.softmax(x.masked_fill(~keep, -math.inf), dim=-1)
            out[t:t + n, h] = torch.where(keep.any(dim=-1, keepdim=True), w @ v[:, g].contiguous(), 0.0)
        t += n
    return out.reshape(s["tokens"], -1)


def _heads64(case, s, x, gamma, pos):
    if gamma is not None:
        x = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / case["dim"] + EPS) * gamma.double()
    half = s["cos"].shape[1]
    j = torch.arange(half, device="cuda")
    first, second = (j, j + half) if case["pairs"] == "halves" else (2 * j, 2 * j + 1)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y
