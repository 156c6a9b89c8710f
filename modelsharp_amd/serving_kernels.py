"""Operators of a step that answers many requests at once, behind the reference's operator
interface (IKernel, KernelRegistry), next to the decoder-layer operators of decoder_kernels:

  PagedAttention    com.microsoft's operator (the reference has no paged cache): rotation of the
                    new queries and keys, their append to the pages, and attention of each
                    request's new tokens over its own; with norms of queries and keys per head
                    as two further inputs
  QkNormRotary      the norms and the rotation alone, before GroupQueryAttention with do_rotary=0
  LoraMatMulNBits   MatMulNBits with low-rank adapters of many requests beside it

Activations are torch tensors on the device (host arrays are uploaded once per call); caches are
device tensors and are written in place. Nothing here computes on the CPU: an input that the
device kernels do not take raises ModelSharpException.
"""
from __future__ import annotations

import numpy as np

from . import native
from .decoder_kernels import _attr_float, _DeviceInputs, _present, _stream, _torch
from .graph import GraphContext, GraphNode, IKernel, KernelRegistry, ModelGraph, ModelSharpException


def _ptr(t):
    return None if t is None else t.data_ptr()


def _optional(node: GraphNode, i: int) -> str:
    return node.inputs[i] if len(node.inputs) > i else ""


def _heads(node: GraphNode, op: str) -> tuple[int, int]:
    H, G = node.attr_int("num_heads", 0), node.attr_int("kv_num_heads", 0)
    if H <= 0 or G <= 0:
        raise ModelSharpException(f"{op} requires positive 'num_heads' and 'kv_num_heads'.")
    if H % G != 0:
        raise ModelSharpException(f"{op} num_heads={H} must be a multiple of kv_num_heads={G}.")
    return H, G


class _Serving(IKernel):
    """A kernel that runs on its first input's device, whatever the current one is."""

    def __init__(self):
        self._dev = _DeviceInputs()

    def execute(self, node: GraphNode, ctx: GraphContext) -> None:
        self._check(node)
        t = ctx.get_tensor(node.inputs[0])
        if isinstance(t, np.ndarray):
            self._run(node, ctx)
        elif t.device.type != "cuda":
            raise ModelSharpException(f"{self.op_type} '{node.inputs[0]}' is a tensor on {t.device}; expected a host "
                                      "array or a device tensor.")
        else:
            with _torch().cuda.device(t.device):
                self._run(node, ctx)

    def _check(self, node):
        """What the attributes alone decide."""

    def _input(self, ctx, name, device):
        """A further fp32 input, on the first one's device wherever it lies."""
        return self._dev.input(ctx, name).to(device)

    def _gamma(self, ctx, name, D, device):
        if not name:
            return None
        g = self._input(ctx, name, device)
        if g.numel() != D:
            raise ModelSharpException(f"{self.op_type} norm weight has {g.numel()} elements; expected head_dim={D}.")
        return g.reshape(-1)

    def _rotary(self, node, ctx, i, device):
        """The cos and sin caches at inputs i and i + 1."""
        if not _optional(node, i) or not _optional(node, i + 1):
            raise ModelSharpException(f"{self.op_type} do_rotary=1 requires cos_cache (input {i}) and sin_cache "
                                      f"(input {i + 1}).")
        cos, sin = (self._input(ctx, node.inputs[j], device) for j in (i, i + 1))
        if cos.dim() != 2 or cos.shape != sin.shape:
            raise ModelSharpException(f"{self.op_type} cos_cache and sin_cache must be equal 2-D shapes.")
        return cos, sin

    def _lengths(self, ctx, name, n, device):
        t = self._dev.i32(ctx.get_tensor(name)).reshape(-1)
        if t.numel() != n:
            raise ModelSharpException(f"{self.op_type} '{name}' has {t.numel()} elements; expected {n}.")
        return t.to(device)


class HipPagedAttentionKernel(_Serving):
    """PagedAttention: query [tokens, num_heads * D] (or packed [tokens, (num_heads + 2 *
    kv_num_heads) * D] with key and value omitted), key, value, key_cache and value_cache
    [num_blocks, block_size, kv_num_heads, D] (fp32 or fp16 device tensors, written in place),
    cumulative_sequence_length [requests + 1], past_seqlens [requests], block_table [requests,
    max_blocks], cos_cache, sin_cache, then q_norm and k_norm weights [D] (optional, with
    attribute epsilon). Rows past the last request's of the output are zeros."""
    op_type = "PagedAttention"

    def _check(self, node):
        _heads(node, self.op_type)
        if _attr_float(node, "softcap", 0.0) != 0.0:
            raise ModelSharpException("PagedAttention softcap is not supported.")

    def _run(self, node: GraphNode, ctx: GraphContext) -> None:
        torch = _torch()
        H, G = _heads(node, self.op_type)
        q = self._dev.input(ctx, node.inputs[0])
        if q.dim() != 2:
            raise ModelSharpException(f"PagedAttention supports only 2-D query [tokens, hidden]; got rank {q.dim()}.")
        T, hidden = int(q.shape[0]), int(q.shape[1])
        packed = not _optional(node, 1)
        if packed != (not _optional(node, 2)):
            raise ModelSharpException("PagedAttention key and value must be given together, or neither with a packed query.")
        unit = H + 2 * G if packed else H
        if hidden % unit != 0:
            raise ModelSharpException(f"PagedAttention query hidden {hidden} not divisible by {unit} heads.")
        D = hidden // unit
        caches = [ctx.get_tensor(node.inputs[i]) for i in (3, 4)]
        for c in caches:
            if isinstance(c, np.ndarray) or c.dim() != 4 or tuple(c.shape[2:]) != (G, D) or not c.is_contiguous() or \
                    c.dtype not in (torch.float32, torch.float16) or c.shape != caches[0].shape or \
                    c.dtype != caches[0].dtype or c.device != q.device:
                raise ModelSharpException("PagedAttention key_cache and value_cache must be contiguous fp32 or fp16 "
                                          "tensors [num_blocks, block_size, kv_num_heads, head_dim] on the query's "
                                          "device.")
        past_src = ctx.get_tensor(node.inputs[6])
        R = int(np.prod(past_src.shape))
        cu_src = ctx.get_tensor(node.inputs[5])
        past = self._lengths(ctx, node.inputs[6], R, q.device)
        cu = self._lengths(ctx, node.inputs[5], R + 1, q.device)
        table = self._dev.i32(ctx.get_tensor(node.inputs[7])).to(q.device)
        if table.dim() != 2 or int(table.shape[0]) != R:
            raise ModelSharpException(f"PagedAttention block_table must be [{R}, max_blocks].")
        d = native.PagedDesc(
            tokens=T, requests=R, num_heads=H, kv_num_heads=G, head_dim=D, page_size=int(caches[0].shape[1]),
            num_pages=int(caches[0].shape[0]), max_pages=int(table.shape[1]),
            cache_type=native.MS_HIP_DTYPE_F16 if caches[0].dtype == torch.float16 else native.MS_HIP_DTYPE_F32,
            local_window_size=node.attr_int("local_window_size", -1), scale=_attr_float(node, "scale", 0.0),
            do_rotary=int(node.attr_int("do_rotary", 0) != 0), eps=_attr_float(node, "epsilon", 1e-6),
            rotary_interleaved=int(node.attr_int("rotary_interleaved", 0) != 0))
        if isinstance(cu_src, np.ndarray) and isinstance(past_src, np.ndarray) and R:
            # lengths the host knows size the launch; those on the device are not fetched for it
            new = np.diff(cu_src.reshape(-1).astype(np.int64))
            d.max_new = max(0, min(int(new.max()), T))
            d.max_total = max(0, min(int((new + past_src.reshape(-1)).max()), 2 ** 30))
        if packed:
            d.q_stride = d.k_stride = d.v_stride = hidden
            pq, pk, pv = q.data_ptr(), q.data_ptr() + 4 * H * D, q.data_ptr() + 4 * (H + G) * D
        else:
            k, v = (self._input(ctx, node.inputs[i], q.device) for i in (1, 2))
            if tuple(k.shape) != (T, G * D) or tuple(v.shape) != (T, G * D):
                raise ModelSharpException(f"PagedAttention key and value must be [{T}, {G * D}].")
            pq, pk, pv = q.data_ptr(), k.data_ptr(), v.data_ptr()
        cos = sin = None
        if d.do_rotary:
            cos, sin = self._rotary(node, ctx, 8, q.device)
            d.cos_rows, d.cos_cols = int(cos.shape[0]), int(cos.shape[1])
        gq, gk = (self._gamma(ctx, _optional(node, i), D, q.device) for i in (10, 11))
        native.paged_attention_check(d)   # before the caches are written
        turned = torch.empty((T, H * D), dtype=torch.float32, device=q.device)
        out = torch.zeros_like(turned)
        st = _stream(q)
        native.paged_append(d, pq, pk, pv, _ptr(gq), _ptr(gk), cu.data_ptr(), past.data_ptr(), table.data_ptr(), _ptr(cos),
                            _ptr(sin), turned.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), st)
        d.q_stride = 0
        n = native.paged_attention_workspace_size(d)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        native.paged_attention(d, turned.data_ptr(), cu.data_ptr(), past.data_ptr(), table.data_ptr(),
                               caches[0].data_ptr(), caches[1].data_ptr(), out.data_ptr(), _ptr(ws), n, st)
        ctx.set(node.outputs[0], out)
        for i in (1, 2):
            if _present(node, i):
                ctx.set(node.outputs[i], caches[i - 1])


class HipQkNormRotaryKernel(_Serving):
    """QkNormRotary(query [..., num_heads * D], key [..., kv_num_heads * D], q_norm, k_norm [D] or
    omitted, position_ids (one for each row), cos_cache, sin_cache) -> (query, key), with
    attributes num_heads, kv_num_heads, epsilon, do_rotary (1 unless given), rotary_interleaved."""
    op_type = "QkNormRotary"

    def _check(self, node):
        _heads(node, self.op_type)

    def _run(self, node: GraphNode, ctx: GraphContext) -> None:
        torch = _torch()
        H, G = _heads(node, self.op_type)
        q = self._dev.input(ctx, node.inputs[0])
        k = self._input(ctx, node.inputs[1], q.device)
        T = int(np.prod(q.shape[:-1]))
        D = int(q.shape[-1]) // H
        if int(q.shape[-1]) != H * D or tuple(k.shape) != tuple(q.shape[:-1]) + (G * D,):
            raise ModelSharpException(f"QkNormRotary query and key must be [..., {H} * head_dim] and [..., {G} * head_dim].")
        d = native.QkNormDesc(tokens=T, num_heads=H, kv_num_heads=G, head_dim=D, eps=_attr_float(node, "epsilon", 1e-6),
                              do_rotary=int(node.attr_int("do_rotary", 1) != 0),
                              rotary_interleaved=int(node.attr_int("rotary_interleaved", 0) != 0))
        pos = cos = sin = None
        if d.do_rotary:
            if not _optional(node, 4):
                raise ModelSharpException("QkNormRotary do_rotary=1 requires position_ids (input 4).")
            pos = self._lengths(ctx, node.inputs[4], T, q.device)
            cos, sin = self._rotary(node, ctx, 5, q.device)
            d.cos_rows, d.cos_cols = int(cos.shape[0]), int(cos.shape[1])
        gq, gk = (self._gamma(ctx, _optional(node, i), D, q.device) for i in (2, 3))
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        native.qk_norm_rotary(d, q.data_ptr(), k.data_ptr(), _ptr(gq), _ptr(gk), _ptr(pos), _ptr(cos), _ptr(sin),
                              qo.data_ptr(), ko.data_ptr(), _stream(q))
        ctx.set(node.outputs[0], qo)
        ctx.set(node.outputs[1], ko)


class HipLoraMatMulNBitsKernel(_Serving):
    """LoraMatMulNBits: MatMulNBits' inputs A, B, scales, zero_points (or omitted), then lora_a
    [adapters, max_rank, K], lora_b [adapters, N, max_rank] (fp32 or fp16), ranks [adapters] and
    lora_scales [adapters] (both optional), adapter_ids (one for each row of A; a row whose id names no
    adapter has the projection alone). Attributes as MatMulNBits."""
    op_type = "LoraMatMulNBits"

    def __init__(self, matmul=None):
        super().__init__()
        from .hip_kernel import HipMatMulNBitsKernel
        self._mm = matmul if matmul is not None else HipMatMulNBitsKernel()
        self._weights: dict[int, tuple] = {}

    def close(self):
        self._mm.close()
        self._weights.clear()

    @staticmethod
    def _projection(node: GraphNode, a: str, y: str) -> GraphNode:
        return GraphNode("MatMulNBits", node.name + "/mm", [a] + list(node.inputs[1:4]), [y], node.attributes)

    def preload(self, graph: ModelGraph) -> int:
        """Load-time upload of the projections' weights (HipMatMulNBitsKernel.preload)."""
        g = ModelGraph([self._projection(n, n.inputs[0], n.outputs[0]) for n in graph.nodes if n.op_type == self.op_type],
                       graph.initializers)
        g.sources = getattr(graph, "sources", {})
        return self._mm.preload(g)

    def _adapter(self, ctx, name, device):
        """A tensor of adapter weights in its own type; initializers are uploaded once and kept."""
        torch = _torch()
        t = ctx.get_tensor(name)
        if t.ndim != 3 or t.dtype not in (torch.float32, torch.float16, np.float32, np.float16):
            raise ModelSharpException(f"LoraMatMulNBits '{name}' must be a 3-D fp32 or fp16 tensor.")
        if isinstance(t, np.ndarray):
            hit = self._weights.get(id(t)) if ctx.is_constant(name) else None
            if hit is not None and hit[0] is t:
                return hit[1].to(device)
            d = torch.from_numpy(np.ascontiguousarray(t)).to(device)
            if ctx.is_constant(name):
                self._weights[id(t)] = (t, d)
            return d
        return t.to(device).contiguous()

    def _run(self, node: GraphNode, ctx: GraphContext) -> None:
        torch = _torch()
        x = self._dev.input(ctx, node.inputs[0])
        mine = GraphContext({**ctx.values, node.inputs[0]: x}, ctx.constants)
        self._mm.execute(self._projection(node, node.inputs[0], node.outputs[0]), mine)
        y = mine.get_tensor(node.outputs[0])
        K, N = int(x.shape[-1]), int(y.shape[-1])
        T = y.numel() // N
        a, b = (self._adapter(ctx, node.inputs[i], x.device) for i in (4, 5))
        A, rank = int(a.shape[0]), int(a.shape[1])
        if int(a.shape[2]) != K or tuple(b.shape) != (A, N, rank) or a.dtype != b.dtype:
            raise ModelSharpException(f"LoraMatMulNBits lora_a must be [adapters, rank, {K}] and lora_b [adapters, {N}, "
                                      "rank] of one type.")
        ranks = self._lengths(ctx, node.inputs[6], A, x.device) if _optional(node, 6) else None
        scales = self._input(ctx, node.inputs[7], x.device).reshape(-1) if _optional(node, 7) else None
        if scales is not None and scales.numel() != A:
            raise ModelSharpException(f"LoraMatMulNBits lora_scales has {scales.numel()} elements; expected {A}.")
        which = self._lengths(ctx, node.inputs[8], T, x.device)
        d = native.LoraDesc(tokens=T, K=K, N=N, adapters=A, max_rank=rank,
                            weight_type=native.MS_HIP_DTYPE_F16 if a.dtype == torch.float16 else native.MS_HIP_DTYPE_F32)
        n = native.lora_workspace_size(d)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)
        native.lora(d, x.data_ptr(), a.data_ptr(), b.data_ptr(), _ptr(ranks), _ptr(scales), which.data_ptr(), y.data_ptr(),
                    y.data_ptr(), ws.data_ptr(), n, _stream(x))
        ctx.set(node.outputs[0], y)


def register_serving_kernels(registry: KernelRegistry) -> KernelRegistry:
    """Registers the device kernels of a serving step (last registration wins,
    KernelRegistry.cs:20-24)."""
    for k in (HipPagedAttentionKernel(), HipQkNormRotaryKernel(), HipLoraMatMulNBitsKernel()):
        registry.register(k)
    return registry
