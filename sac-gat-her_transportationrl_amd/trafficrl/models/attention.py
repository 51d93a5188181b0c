"""Softmax attention between the nodes of each network of a packed batch, on
gfx950 kernels (csrc/node_attention.hip): the global counterpart of GATConv's
attention over a node's in-edges (src/models/gat_encoder.py:22-25)."""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib
from ..autograd import no_tangents, once


def _strided(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it (channels contiguous, rows and
    heads 16-byte aligned), else a contiguous copy."""
    unit = 16 // t.element_size()
    for dim in (1, 0):   # a dimension of one may have any stride, and contiguous() would leave it
        if t.shape[dim] == 1 and t.stride(dim) % unit:
            t = t.squeeze(dim).unsqueeze(dim)
    s = t.stride()
    if s[2] == 1 and s[0] % unit == 0 and s[1] % unit == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _args(q, k, v, ptr, k_ptr, dist, slope, rest, out, low, lse, backward: bool, grads=(0, 0, 0, 0, 0)):
    """The argument block and the workspace it points to."""
    scale, cap, max_queries, max_nodes, code = rest
    rows, heads, channels = q.shape
    nodes, kv_heads, _ = k.shape
    q_row, q_head, _ = q.stride()
    k_row, k_head, _ = k.stride()
    v_row, v_head, _ = v.stride()
    d = (0, 0, 0, 0, 0, 0)
    if dist is not None:
        # an empty matrix shows no pair, which a null pointer would not say
        d = (*dist.shape[-2:], dist.data_ptr() or ptr.data_ptr(), dist.stride(0) if dist.dim() == 3 else 0, dist.stride(-2),
             0 if slope is None else slope.data_ptr())
    a = _lib.TrxNodeAttentionArgs(
        ptr.numel() - 1, heads, kv_heads, channels, code, d[0], d[1], scale, cap, max_queries, max_nodes, rows, nodes,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_row, q_head, k_row, k_head, v_row, v_head, ptr.data_ptr(),
        k_ptr.data_ptr(), *d[2:], out.data_ptr(), 0 if low is None else low.data_ptr(),
        0 if lse is None else lse.data_ptr(), *grads)
    need = _lib.load().trx_node_attention_workspace_bytes(a, backward)
    ws = None
    if need > 0:
        ws = torch.empty(need, device=q.device, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    return a, ws


def _launch(q, k, v, ptr, k_ptr, dist, slope, rest, save: bool):
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = low = None
    if save:
        lse = torch.empty(q.shape[:2], device=q.device, dtype=torch.float32)
        low = torch.empty_like(out) if out.dtype != torch.float32 else None
    a, ws = _args(q, k, v, ptr, k_ptr, dist, slope, rest, out, low, lse, False)
    _lib.check(_lib.load().trx_node_attention_forward(a, _lib.raw_stream(q.device)), "trx_node_attention_forward")
    return out, low, lse


def _launch_backward(q, k, v, slope, ptr, k_ptr, dist, out, low, lse, rest, grad_out, wants_slope):
    grad_out = grad_out.contiguous()
    if grad_out.data_ptr() % 16:
        grad_out = grad_out.clone()
    gq, gk, gv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
    gs = torch.empty_like(slope) if wants_slope else None
    a, ws = _args(q, k, v, ptr, k_ptr, dist, slope, rest, out, low, lse, True,
                  (grad_out.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), 0 if gs is None else gs.data_ptr()))
    _lib.check(_lib.load().trx_node_attention_backward(a, _lib.raw_stream(q.device)), "trx_node_attention_backward")
    return gq, gk, gv, gs


class _NodeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slope, ptr, k_ptr, dist, rest):
        out, low, lse = _lib.on_device(q.device, _launch, q, k, v, ptr, k_ptr, dist, slope, rest, True)
        ctx.save_for_backward(q, k, v, slope, ptr, k_ptr, dist, out, low, lse)
        ctx.rest = rest
        return out

    @staticmethod
    @once("node_attention")
    def backward(ctx, grad_out):
        return *_lib.on_device(grad_out.device, _launch_backward, *ctx.saved_tensors, ctx.rest, grad_out,
                               ctx.needs_input_grad[3]), None, None, None, None


def node_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ptr: torch.Tensor, *,
                   k_ptr: Optional[torch.Tensor] = None, dist: Optional[torch.Tensor] = None,
                   slope: Optional[torch.Tensor] = None, scale: Optional[float] = None, cap: float = 0.0,
                   max_queries: Optional[int] = None, max_nodes: Optional[int] = None) -> torch.Tensor:
    """out[i, h] = sum_j softmax_j(z_ij - slope[h] d_ij) v[j, h'] over the nodes j
    of row i's own network, z = scale <q[i, h], k[j, h']>, capped to cap tanh(z /
    cap) where cap > 0.

    q [rows, heads, channels], k and v [nodes, kv_heads, channels]: one of
    float32, bfloat16, float16; any row and head strides; head h reads key/value
    head h' = h // (heads / kv_heads).  channels: a multiple of 8 up to 128.
    ptr: int64 [networks + 1], the first row of each network in q (PyG's
    Batch.ptr); k_ptr: the same for k and v where the queries are not the nodes
    themselves (one decision query per network, say).
    dist: float32 travel times, [n, n] for all networks or [networks, n, n] (the
    top left corner of n x n for smaller ones; [.., queries, nodes] with k_ptr);
    a pair that is not finite, or outside the matrix, is not seen.  slope:
    float32 [heads], what a unit of distance costs; without it dist only masks.
    scale: 1 / sqrt(channels) unless given.
    A row that sees no node gives zeros and passes no gradient.  Entries of q,
    k, v and the gradient must be finite, or a network's own rows (no other
    network's) may become NaN.  max_queries / max_nodes: the largest network's
    rows; hints that shape the launch, taken from dist's shape where it is given.
    Without either, a batch of many small networks takes several times as long.

    Differentiable once in q, k, v and slope (a forward-mode tangent is refused).
    Scores, softmax statistics and sums are float32; with half types the
    probabilities and the scores' gradients are rounded to the type where they
    enter a matrix product.  Results do not depend on timing: no float atomics.
    Asynchronous on the current stream and capturable; before a backward pass is captured, drop
    the eager graphs of the same leaves (autograd ties a leaf's accumulation to
    the stream of its first live graph)."""
    what = "node_attention"
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k, v must be [rows, heads, channels], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    code = _lib.float_code(q, f"{what}: q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k, v differ in type: {q.dtype}, {k.dtype}, {v.dtype}")
    rows, H, C = q.shape
    nodes, kv_heads, channels = k.shape
    if k.shape != v.shape or channels != C:
        raise ValueError(f"{what}: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not fit together")
    if H < 1 or kv_heads < 1 or H % kv_heads:
        raise ValueError(f"{what}: {kv_heads} key/value heads must divide {H} heads")
    if C < 8 or C % 8 or C > _lib.ATT_MAX_CHANNELS:
        raise ValueError(f"{what}: channels must be a multiple of 8 up to {_lib.ATT_MAX_CHANNELS}, got {C}")
    if k_ptr is None:
        if rows != nodes:
            raise ValueError(f"{what}: {rows} query rows and {nodes} nodes need a k_ptr")
        k_ptr = ptr
    for p in (ptr,) if k_ptr is ptr else (ptr, k_ptr):
        if p.dtype != torch.int64 or p.dim() != 1 or p.numel() != ptr.numel() or p.numel() < 1:
            raise ValueError(f"{what}: ptr and k_ptr must be int64 [networks + 1]")
    if dist is not None:
        if dist.dtype != torch.float32 or dist.dim() not in (2, 3):
            raise ValueError(f"{what}: dist must be float32 [n, n] or [networks, n, n]")
        if dist.dim() == 3 and dist.shape[0] != ptr.numel() - 1:
            raise ValueError(f"{what}: {dist.shape[0]} distance matrices for {ptr.numel() - 1} networks")
        if dist.requires_grad:
            raise ValueError(f"{what}: dist has no gradient (detach it)")
    if slope is not None:
        if dist is None:
            raise ValueError(f"{what}: slope needs dist")
        if slope.dtype != torch.float32 or slope.shape != (H,):
            raise ValueError(f"{what}: slope must be float32 [{H}]")
    scale = 1.0 / math.sqrt(C) if scale is None else float(scale)
    cap = float(cap)
    if not math.isfinite(scale) or not math.isfinite(cap) or cap < 0.0:
        raise ValueError(f"{what}: scale must be finite, cap finite and >= 0 (got {scale}, {cap})")
    if cap > 0.0 and not abs(scale) < cap * 1e30:
        raise ValueError(f"{what}: cap {cap} is too small beside scale {scale}")
    # the distances' shape bounds the largest network; a single one is bounded by its rows
    most_q, most_k = dist.shape[-2:] if dist is not None and ptr.numel() > 2 else (rows, nodes)
    max_queries = min(rows, most_q) if max_queries is None else int(max_queries)
    max_nodes = min(nodes, most_k) if max_nodes is None else int(max_nodes)
    if max_queries < 0 or max_nodes < 0:
        raise ValueError(f"{what}: max_queries and max_nodes must be >= 0")
    no_tangents(what, q, k, v, dist, slope)
    _lib.same_device(what, q, k, v, ptr, k_ptr, dist, slope)
    q, k, v, ptr, k_ptr = _strided(q), _strided(k), _strided(v), ptr.contiguous(), k_ptr.contiguous()
    if dist is not None and dist.stride(-1) != 1:
        dist = dist.contiguous()
    if slope is not None:
        slope = slope.contiguous()
    rest = scale, cap, max_queries, max_nodes, code
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (slope is not None and slope.requires_grad)):
        return _NodeAttention.apply(q, k, v, slope, ptr, k_ptr, dist, rest)
    return _lib.on_device(q.device, _launch, q, k, v, ptr, k_ptr, dist, slope, rest, False)[0]
