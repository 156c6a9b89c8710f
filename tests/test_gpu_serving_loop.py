"""A server's loop on the GPU: plan, append, attention behind a shared prefix, projection, sampling and commit as
one captured graph and as nodes of the engine, each operator checked on what it was given."""
from __future__ import annotations

import numpy as np
import pytest

import loop_ref
import serving_ref as ref
from modelsharp_amd import native
from test_gpu_serving import check_attention, dev, log, ptr

pytestmark = pytest.mark.gpu
F16, F32, I32 = np.float16, np.float32, np.int32

R, H, G, D, PAGE, WIDTH, PAGES, S, V, CHUNK, LONGEST = 12, 8, 2, 64, 16, 200, 150, 70, 1009, 5, 40
END = 7   # a token that is this modulo 8 ends its request


class Server:
    """Buffers of a loop over R requests that all begin with the same S positions: whole pages of them are shared,
    the rest of the last page is each request's own copy."""

    def __init__(self, seed, dtype):
        import torch
        rng = self.rng = np.random.default_rng(seed)
        self.dtype, self.end, self.prefix = dtype, END, S
        whole = S // PAGE
        order = rng.permutation(PAGES).astype(I32)
        table = np.full((R, WIDTH), -1, I32)
        table[:, :whole] = order[:whole]
        table[:, whole] = order[whole:whole + R]
        free = np.full(PAGES, -1, I32)
        count = PAGES - whole - R
        free[:count] = order[whole + R:]
        kc, vc = (rng.standard_normal((PAGES, PAGE, G, D)).astype(dtype) for _ in range(2))
        for r in range(1, R):
            for c in (kc, vc):
                c[table[r, whole], :S % PAGE] = c[table[0, whole], :S % PAGE]
        self.prompts = rng.integers(1, 14, R)
        ids = rng.integers(8, V, (R, LONGEST + 1))
        known = S + self.prompts      # positions whose token is known
        self.embed = torch.from_numpy(rng.standard_normal((V, (H + 2 * G) * D)).astype(F32)).cuda()
        self.out_w = torch.from_numpy((rng.standard_normal((H * D, V)) * 0.2).astype(F32)).cuda()
        self.tokens = T = R * CHUNK - 25   # not enough for everyone's chunk
        names = dict(table=table, past=np.full(R, S), free=free, count=[count], ids=ids, known=known, first=known,
                     cu=np.zeros(R + 1), used=[0], rows_r=np.zeros(T), rows_p=np.zeros(T), rows_s=np.zeros(T),
                     groups=[0, R], shared=[S], done=np.zeros(R), keep=np.full(R, whole), want=np.zeros(R),
                     drawn=np.zeros(R), k=rng.choice([0, 3, 40], R))
        for name, x in names.items():
            setattr(self, name, dev(np.asarray(x, np.int64 if name in ("ids", "known", "first") else I32)))
        self.kc, self.vc = dev(kc), dev(vc)
        self.t, self.p, self.m = (dev(x.astype(F32)) for x in (rng.uniform(0.5, 1.5, R), rng.uniform(0.6, 1.0, R),
                                                               rng.uniform(0.0, 0.05, R)))
        self.t[3] = 0.0
        self.u = dev(np.zeros(R, F32))
        self.q = torch.zeros(T, H * D, device="cuda")
        self.attn = torch.zeros(T, H * D, device="cuda")
        self.logits = torch.zeros(R, V, device="cuda")
        self.lp = torch.zeros(R, device="cuda")
        self.step_desc = native.StepDesc(tokens=T, requests=R, page_size=PAGE, num_pages=PAGES, max_pages=WIDTH)
        cols = (H + 2 * G) * D
        self.paged = native.PagedDesc(tokens=T, requests=R, num_heads=H, kv_num_heads=G, head_dim=D, page_size=PAGE,
                                      num_pages=PAGES, max_pages=WIDTH, q_stride=cols, k_stride=cols, v_stride=cols,
                                      cache_type=native.MS_HIP_DTYPE_F16 if dtype == F16 else native.MS_HIP_DTYPE_F32,
                                      local_window_size=-1)
        self.attend = native.PagedDesc.from_buffer_copy(self.paged)
        self.attend.q_stride = 0
        self.share = native.SharedDesc(groups=1)
        # by the table's width: the call shares
        assert (R - 1) * WIDTH * PAGE * 2 * G * D * np.dtype(dtype).itemsize >= 16 << 20
        self.n_attn = native.paged_shared_attention_workspace_size(self.attend, self.share)
        self.ws_attn = torch.empty(self.n_attn, dtype=torch.uint8, device="cuda")
        self.sampled = native.SampleDesc(rows=R, vocab=V)
        self.n_samp = native.sample_workspace_size(self.sampled)
        self.ws_samp = torch.empty(self.n_samp, dtype=torch.uint8, device="cuda")

    def step(self, st):
        """A step of the loop: nothing here waits for the device or reads a length on the host."""
        import torch
        self.want.copy_((self.known - self.past).clamp(0, CHUNK))
        native.paged_plan(self.step_desc, *map(ptr, (self.want, self.past, self.free, self.count, self.table, self.cu,
                                                     self.used, self.rows_r, self.rows_p, self.rows_s)), st)
        here = self.rows_r >= 0
        ids = self.ids[self.rows_r.clamp(min=0).long(), (self.rows_p - S).clamp(0, LONGEST).long()]
        x = self.embed[torch.where(here, ids, 0)]
        step = 4 * D
        native.paged_append(self.paged, x.data_ptr(), x.data_ptr() + H * step, x.data_ptr() + (H + G) * step, None, None,
                            *map(ptr, (self.cu, self.past, self.table)), None, None, *map(ptr, (self.q, self.kc, self.vc)), st)
        native.paged_shared_attention(self.attend, self.share, *map(ptr, (
            self.q, self.cu, self.past, self.table, self.groups, self.shared, self.kc, self.vc, self.attn, self.ws_attn)),
            self.n_attn, st)
        last = (self.cu[1:] - 1).clamp(min=0).long()
        self.logits.copy_(self.attn[last] @ self.out_w)
        native.sample(self.sampled, *map(ptr, (self.logits, self.t, self.k, self.p, self.m, self.u, self.drawn, self.lp,
                                               self.ws_samp)), self.n_samp, st)
        served = self.cu[1:] > self.cu[:-1]
        total = self.past + torch.where(served, self.cu[1:] - self.cu[:-1], 0)
        draws = served & (total == self.known)       # the prompt is through: the row's token is the next one
        at = (total - S).clamp(0, LONGEST).long()[:, None]
        self.ids.scatter_(1, at, torch.where(draws, self.drawn.long(), self.ids.gather(1, at)[:, 0])[:, None])
        self.known.add_(draws.long())
        self.done.copy_(draws & ((self.drawn % 8 == self.end) | (self.known > S + LONGEST)))
        native.paged_commit(self.step_desc, *map(ptr, (self.cu, self.used, self.done, self.keep, self.past, self.table,
                                                       self.free, self.count)), st)

    def restart(self):
        """The requests that have ended begin anew behind the prefix, their part of its last page in a new page."""
        import torch
        done = self.done != 0
        n = int(done.sum())
        if not n:
            return
        count = int(self.count)
        pages = self.free[count - n:count].clone()
        self.count -= n
        which = torch.nonzero(done)[:, 0]
        self.table[which, S // PAGE] = pages
        source = self.copy_of_the_end
        for c, x in zip((self.kc, self.vc), source):
            c[pages.long(), :S % PAGE] = x
        self.past[which], self.known[which] = S, self.first[which]

    def snapshot(self):
        return {n: getattr(self, n).cpu().numpy().copy() for n in (
            "table", "past", "free", "count", "cu", "used", "rows_r", "rows_p", "rows_s", "want", "done", "drawn", "lp", "logits",
            "q", "attn", "kc", "vc", "u", "t", "k", "p", "m", "known")}


def check_step(s, before, after):
    """Each operator's results on its own inputs, in 64 bits."""
    T = s.tokens
    want = np.clip(before["known"] - before["past"], 0, CHUNK)
    exp = loop_ref.plan(want, before["past"], before["free"], before["count"][0], before["table"], T, PAGE, PAGES)
    for name, e in zip(("cu", "used", "rows_r", "rows_p", "rows_s"), exp):
        assert np.array_equal(after[name].reshape(np.shape(e)), e), name
    cu, table = exp[0], exp[5]
    b = ref.Batch(0, np.diff(cu), before["past"], G, D, PAGE, s.dtype)
    b.num_pages, b.max_pages, b.table, b.k, b.v, b.tokens = PAGES, WIDTH, table, after["kc"], after["vc"], int(cu[-1])
    check_attention(after["attn"][:b.tokens], b, after["q"][:b.tokens], H)
    assert not after["attn"][b.tokens:].any()   # rows behind the last request's
    for t, r, pos in b.each_token():
        assert b.row(r, pos) == after["rows_s"][t]
    for r in np.flatnonzero(np.diff(cu)):
        args = [after[n][r] for n in ("t", "k", "p", "m", "u")]
        token, lp, tol = loop_ref.sample(after["logits"][r], *args)
        if not loop_ref.near_a_border(after["logits"][r], *args):
            assert after["drawn"][r] == token and abs(after["lp"][r] - lp) <= tol
    got = loop_ref.commit(cu, exp[1], after["done"], np.full(R, S // PAGE), before["past"], table, before["free"],
                          before["count"][0], PAGE, PAGES)
    for name, e in zip(("past", "table", "free", "count"), got):
        assert np.array_equal(after[name].reshape(np.shape(e)), e), name
    held = after["table"][after["table"] >= 0]
    own = np.concatenate([np.unique(after["table"][:, :S // PAGE]), after["table"][:, S // PAGE:][after["table"][:, S // PAGE:] >= 0]])
    free = after["free"][:after["count"][0]]
    assert len(held) and len(own) + len(free) == PAGES and len(np.unique(np.concatenate([own, free]))) == PAGES   # none lost


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_loop_replayed_from_a_graph(gpu, dtype):
    """Captured once. Prompts in chunks, single tokens, requests that wait for rows, end and begin anew."""
    import torch
    s = Server(5, dtype)
    end = int(s.table[0, S // PAGE])
    s.copy_of_the_end = [c[end, :S % PAGE].clone() for c in (s.kc, s.vc)]
    known = s.known.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.known.copy_(s.past)          # nothing is wanted: nothing changes
        s.step(side.cuda_stream)
        side.synchronize()
        assert int(s.cu[-1]) == 0 and int(s.count) == PAGES - S // PAGE - R and not s.attn.any()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.step(side.cuda_stream)
    s.known.copy_(known)
    ended = waited = 0
    for i in range(24):
        s.u.copy_(dev(s.rng.random(R).astype(F32)))
        s.attn.zero_()
        torch.cuda.synchronize()
        before = s.snapshot()
        graph.replay()
        torch.cuda.synchronize()
        after = s.snapshot()
        log(f"replay {i}: rows {after['cu'][-1]}, ended {after['done'].sum()}, free {after['count'][0]}")
        check_step(s, before, after)
        waited += int((np.diff(after["cu"]) < after["want"]).sum())
        ended += int((after["done"] != 0).sum())
        s.restart()
    assert ended and waited


def test_two_loops_on_two_streams(gpu):
    """Each with buffers and workspaces of its own, their steps in flight at once; as each alone."""
    import torch
    runs = []
    for both in (False, True):
        servers = [Server(6 + i, (F16, F32)[i]) for i in range(2)]
        for s in servers:
            s.end = 8   # (none ends)
        streams = [torch.cuda.Stream() for _ in servers]
        us = [[dev(s.rng.random(R).astype(F32)) for _ in range(6)] for s in servers]
        torch.cuda.synchronize()
        for order in ([(i, s, st) for i in range(6) for s, st in zip((0, 1), streams)] if both else
                      [(i, s, streams[s]) for s in (0, 1) for i in range(6)]):
            i, which, st = order
            with torch.cuda.stream(st):
                servers[which].u.copy_(us[which][i])
                servers[which].step(st.cuda_stream)
        torch.cuda.synchronize()
        runs.append([s.snapshot() for s in servers])
        log(f"together {both}")
    for a, b in zip(*runs):
        for name in a:
            assert np.array_equal(a[name], b[name]), name


# ---- graph nodes ----------------------------------------------------------------------------------

@pytest.mark.parametrize("on", ["device", "host"])
def test_nodes_of_a_loop(gpu, on):
    """PagedStepPlan -> PagedAttention behind a shared prefix -> MatMulNBits -> SampleTokens -> PagedStepCommit, run
    by the engine for a few steps."""
    import torch
    from modelsharp_amd import pipeline, workloads
    from modelsharp_amd.graph import GraphNode, ModelGraph
    s = Server(9, F16)
    vocab = 512
    w, sc, z = workloads.make_weights(workloads.Op("head", H * D, vocab, 32, True), seed=3)
    init = {"w": w, "sc": sc, "z": z}
    nodes = [
        GraphNode("PagedStepPlan", "plan", ["table", "past", "free", "count", "want"], ["cu", "rr", "rp", "rs", "used"],
                  {"tokens": R, "block_size": PAGE}),
        GraphNode("PagedAttention", "attn", ["x", "", "", "kc", "vc", "cu", "past", "table", "", "", "", "", "groups", "shared"],
                  ["attn"], {"num_heads": H, "kv_num_heads": G}),
        GraphNode("MatMulNBits", "head", ["attn", "w", "sc", "z"], ["logits"],
                  {"K": H * D, "N": vocab, "bits": 4, "block_size": 32}),
        GraphNode("SampleTokens", "sample", ["logits", "u", "t", "k", "p", "m"], ["next", "lp"]),
        GraphNode("PagedStepCommit", "commit", ["table", "past", "free", "count", "cu", "used", "done", "keep"],
                  ["table2", "past2", "free2", "count2"], {"block_size": PAGE}),
    ]
    engine = pipeline.build(ModelGraph(nodes, init, [], ["cu", "rr", "rp", "rs", "used", "attn", "logits", "next", "lp",
                                                         "table2", "past2", "free2", "count2"]))
    for i in range(4):
        want = np.ones(R, I32)
        want[i::4] = 0
        done = (s.rng.random(R) < 0.2).astype(I32)
        x = s.rng.standard_normal((R, (H + 2 * G) * D)).astype(F32)
        feeds = dict(x=x, want=want, done=done, keep=np.full(R, S // PAGE, I32), u=s.rng.random(R).astype(F32),
                     groups=np.array([0, R], I32), shared=np.array([s.prefix], I32), k=s.k.cpu().numpy(),
                     **{n: getattr(s, n).cpu().numpy() for n in "tpm"})
        if on == "device":
            feeds = {n: dev(v) for n, v in feeds.items()}
        feeds.update({n: getattr(s, n) for n in ("table", "past", "free", "count", "kc", "vc")})
        before = s.snapshot()
        out = {n: v.cpu().numpy() for n, v in engine.run(feeds).items()}
        log(f"nodes step {i}: {int(out['cu'][-1])} rows")
        exp = loop_ref.plan(want, before["past"], before["free"], before["count"][0], before["table"], R, PAGE, PAGES)
        for name, e in zip(("cu", "used", "rr", "rp", "rs"), exp):
            assert np.array_equal(out[name].reshape(np.shape(e)), e), name
        b = ref.Batch(0, np.diff(exp[0]), before["past"], G, D, PAGE, F16)
        b.num_pages, b.max_pages, b.table, b.tokens = PAGES, WIDTH, exp[5], int(exp[0][-1])
        b.k, b.v = s.kc.cpu().numpy(), s.vc.cpu().numpy()
        check_attention(out["attn"][:b.tokens], b, np.ascontiguousarray(x[:b.tokens, :H * D]), H)
        assert not out["attn"][b.tokens:].any()
        for r in range(b.tokens):
            args = [before[n][r] for n in "tkpm"] + [feeds["u"][r] if on == "host" else float(feeds["u"][r])]
            token, lp, tol = loop_ref.sample(out["logits"][r], *args)
            assert loop_ref.near_a_border(out["logits"][r], *args) or (
                out["next"][r] == token and abs(out["lp"][r] - lp) <= tol)
        got = loop_ref.commit(exp[0], exp[1], done, np.full(R, S // PAGE), before["past"], exp[5], before["free"],
                              before["count"][0], PAGE, PAGES)
        for name, e in zip(("past", "table", "free", "count"), got):
            assert np.array_equal(out[name + "2"].reshape(np.shape(e)), e), name
            assert np.array_equal(getattr(s, name).cpu().numpy().reshape(np.shape(e)), e), name   # in place
        for r in np.flatnonzero(done):   # these begin anew behind the prefix's whole pages
            s.past[int(r)] = s.prefix = S // PAGE * PAGE


def test_sample_node_takes_leading_axes_and_optional_inputs(gpu):
    import torch
    from modelsharp_amd.graph import GraphContext, GraphNode
    from modelsharp_amd.serving_kernels import HipSampleTokensKernel
    rng = np.random.default_rng(1)
    x, u = rng.standard_normal((2, 3, 700)).astype(F16), rng.random(6).astype(F32)
    for feed in (x.astype(F32), dev(x)):
        ctx = GraphContext({"x": feed, "u": u, "k": np.array([1, 5, 0, 9, 700, 800], np.int64)})
        HipSampleTokensKernel().execute(GraphNode("SampleTokens", "s", ["x", "u", "", "k"], ["y"]), ctx)
        y = ctx.get_tensor("y")
        assert tuple(y.shape) == (2, 3) and y.dtype == torch.int32
        for r in range(6):
            assert int(y.reshape(-1)[r]) == loop_ref.sample(x.reshape(6, 700)[r].astype(F32), 1.0, [1, 5, 0, 9, 700, 800][r],
                                                            1.0, 0.0, u[r])[0]
    ctx = GraphContext({"x": torch.zeros(0, 50, device="cuda"), "u": np.zeros(0, F32)})
    HipSampleTokensKernel().execute(GraphNode("SampleTokens", "s", ["x", "u"], ["y", "lp"]), ctx)
    assert ctx.get_tensor("y").shape == ctx.get_tensor("lp").shape == (0,)
