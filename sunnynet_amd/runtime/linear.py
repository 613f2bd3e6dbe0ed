"""Linear attention with a decay for each head on the GPU: a matrix state per head, as
prompts and training run it (in chunks) and token by token. The delta rule's recurrence
without its correction; no counterpart in the reference.

Per sequence and value head, with ``a = exp(g)``:

    S_t = a_t S_{t-1} + k_t v_t^T
    out_t = scale S_t^T q_t

``g`` holds a decay per token and head, or one per head. Value head ``h`` of ``H`` reads
query and key head ``h // (H // Hk)``. States and sums are fp32 whatever the inputs' type.
``g <= 0`` is meant; ``-inf`` forgets the state exactly. A value that is not finite makes
its sequence and head NaN from the chunk of up to 64 tokens that holds it on.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .delta import (DTYPES, MAX_HEADS, MAX_K, MAX_STRIDE, MAX_V, _check_state, _ptr, _rows, note_leaves,
                    refuse_tangents)

__all__ = ["LinearAttention", "linear_attention", "linear_bwd", "linear_fwd", "linear_step"]

STEP_TOKENS = 12               # at most this many tokens run token by token
_ARGS = struct.Struct("6P9q9qd1P")     # SnHipLinear
_GRAD = struct.Struct("9P")            # SnHipLinearGrad


def _shapes(q, k, v, g, s0, cu, step=False):
    """(B, T, N, Hk, H, K, V) of a call, after its checks. step: one token, without T axes."""
    names = "q, k (B,Hk,K); v (B,H,V); g (B,H) or (H)" if step else "q, k (B,T,Hk,K); v (B,T,H,V); g (B,T,H) or (H)"
    rank = 3 if step else 4
    if q.dim() != rank or v.dim() != rank or k.shape != q.shape or v.shape[:-2] != q.shape[:-2] \
            or g.shape != v.shape[:-1] and g.shape != v.shape[-2:-1]:
        raise ValueError(f"shape mismatch: {names}")
    B, T = (q.shape[0], 1) if step else q.shape[:2]
    Hk, K = q.shape[-2:]
    H, V = v.shape[-2:]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{H} value heads cannot share {Hk} query and key heads evenly")
    if not 1 <= K <= MAX_K or not 1 <= V <= MAX_V or H > MAX_HEADS:
        raise ValueError(f"head sizes up to K = {MAX_K}, V = {MAX_V} and up to {MAX_HEADS} heads: "
                         f"got K = {K}, V = {V}, {H} heads")
    if H * max(K, V) >= MAX_STRIDE // 2:
        raise ValueError(f"H * K and H * V must be below {MAX_STRIDE // 2}")
    if B * T >= 1 << 30:
        raise ValueError("B * T must be below 2^30")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be float32, bfloat16 or float16, all three the same")
    if g.dtype != torch.float32:
        raise ValueError("g must be float32")
    N = B
    if cu is not None:
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 2 or not cu.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous int32 vector of at least two edges")
        if B != 1:
            raise ValueError("with cu_seqlens the sequences lie end to end in one batch entry: B must be 1")
        N = cu.shape[0] - 1
    if N > 65535:
        raise ValueError("at most 65535 sequences per call")
    if s0 is not None:
        _check_state(s0, (N, H, K, V), "s0")
    dev = q.device
    if not q.is_cuda or k.device != dev or v.device != dev or g.device != dev \
            or s0 is not None and s0.device != dev or cu is not None and cu.device != dev:
        raise ValueError("linear attention takes tensors of one GPU")
    return B, T, N, Hk, H, K, V


def _pack(q, k, v, g, s0, cu, dims, scale, parts=None):
    return _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), _ptr(s0), _ptr(cu), *q.stride()[:3],
                      *k.stride()[:3], *v.stride()[:3], *dims, DTYPES[q.dtype], g.dim() == 1, scale, _ptr(parts))


def linear_fwd(q, k, v, g, s0=None, *, scale=None, cu_seqlens=None, keep=False):
    """q, k (B,T,Hk,K), v (B,T,H,V), g (B,T,H) or (H), s0 (B,H,K,V) or None ->
    (out (B,T,H,V), send (B,H,K,V), parts), without autograd. The last axes of q, k and
    v are contiguous or copied; their other strides are free. With ``cu_seqlens`` (N + 1
    int32 edges on the device, not decreasing) B is 1, sequence n holds tokens
    ``[cu[n], cu[n+1])``, s0 and send are (N,H,K,V), and tokens of no sequence give 0.
    ``parts``: with ``keep`` what linear_bwd needs besides (None for short sequences).
    ``scale``: K ** -0.5 if None."""
    q, k, v, g = _rows(q), _rows(k), _rows(v), g.contiguous()
    dims = _shapes(q, k, v, g, s0, cu_seqlens)
    return _fwd(q, k, v, g, s0, cu_seqlens, dims, scale, keep)


def _fwd(q, k, v, g, s0, cu_seqlens, dims, scale, keep):
    B, T, N, Hk, H, K, V = dims
    scale = K ** -0.5 if scale is None else float(scale)
    out = torch.empty(B, T, H, V, dtype=v.dtype, device=q.device)
    send = torch.empty(N, H, K, V, dtype=torch.float32, device=q.device)
    if B * T == 0 or N == 0:
        send.zero_() if s0 is None else send.copy_(s0)
        return out, send, None
    L = _native.lib()
    if not keep and cu_seqlens is None and T <= STEP_TOKENS:
        rc = _native.on_device(q.device, L.snhip_op_linear_step_dev, _pack(q, k, v, g, s0, None, dims, scale),
                               out.data_ptr(), send.data_ptr())
        _native.check(rc, "snhip_op_linear_step_dev")
        return out, send, None
    floats = L.snhip_op_linear_parts_floats(_pack(q, k, v, g, s0, cu_seqlens, dims, scale))
    parts = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    rc = _native.on_device(q.device, L.snhip_op_linear_fwd_dev, _pack(q, k, v, g, s0, cu_seqlens, dims, scale, parts),
                           out.data_ptr(), send.data_ptr())
    _native.check(rc, "snhip_op_linear_fwd_dev")
    return out, send, parts if keep else None


def linear_bwd(q, k, v, g, s0, send, parts, dout, dsend=None, *, scale=None, cu_seqlens=None, need_ds0=True):
    """Gradients of linear_fwd(..., keep=True), from its send and parts -> (dq, dk, dv, dg,
    ds0): dout (B,T,H,V) of the inputs' type, dsend (N,H,K,V) float32 or None (zeros); dg
    as g; ds0 is None unless ``need_ds0``. The same calls give the same bits."""
    q, k, v, g = _rows(q), _rows(k), _rows(v), g.contiguous()
    dims = _shapes(q, k, v, g, s0, cu_seqlens)
    B, T, N, Hk, H, K, V = dims
    if dout.shape != (B, T, H, V) or dout.dtype != v.dtype or dout.device != q.device:
        raise ValueError("dout must be (B,T,H,V), of the inputs' type and device")
    _check_state(send, (N, H, K, V), "send")
    if dsend is not None:
        _check_state(dsend, (N, H, K, V), "dsend")
    if any(t is not None and t.device != q.device for t in (send, dsend)):
        raise ValueError("linear attention takes tensors of one GPU")
    if B * T and N:
        floats = _native.lib().snhip_op_linear_parts_floats(_pack(q, k, v, g, s0, cu_seqlens, dims, 1.0))
        if (floats > 0) != (parts is not None) or floats and (
                parts.shape != (floats,) or parts.dtype != torch.float32 or parts.device != q.device
                or not parts.is_contiguous()):
            raise ValueError("parts must be linear_fwd's, of the same shapes, with keep=True")
    return _bwd(q, k, v, g, s0, cu_seqlens, dims, scale, send, parts, dout.contiguous(), dsend, need_ds0)


def _bwd(q, k, v, g, s0, cu_seqlens, dims, scale, send, parts, dout, dsend, need_ds0):
    B, T, N, Hk, H, K, V = dims
    scale = K ** -0.5 if scale is None else float(scale)
    dq, dk = (torch.empty(B, T, Hk, K, dtype=q.dtype, device=q.device) for _ in range(2))
    dv = torch.empty(B, T, H, V, dtype=q.dtype, device=q.device)
    dg = torch.empty(g.shape, dtype=torch.float32, device=q.device)
    ds0 = torch.empty(N, H, K, V, dtype=torch.float32, device=q.device) if need_ds0 else None
    if B * T == 0 or N == 0:
        dg.zero_()
        if need_ds0:
            ds0.zero_() if dsend is None else ds0.copy_(dsend)
        return dq, dk, dv, dg, ds0
    L = _native.lib()
    args = _pack(q, k, v, g, s0, cu_seqlens, dims, scale, parts)
    ws = torch.empty(L.snhip_op_linear_bwd_floats(args), dtype=torch.float32, device=q.device)
    grads = _GRAD.pack(dout.data_ptr(), _ptr(dsend), send.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                       dg.data_ptr(), _ptr(ds0), ws.data_ptr())
    rc = _native.on_device(q.device, L.snhip_op_linear_bwd_dev, args, grads)
    _native.check(rc, "snhip_op_linear_bwd_dev")
    return dq, dk, dv, dg, ds0


class LinearAttention(torch.autograd.Function):
    """Linear attention under autograd: (out, send) of linear_fwd, gradients of linear_bwd.
    Keeps the inputs, send, and of long sequences the states that their parts begin with
    (snhip_op_linear_parts_floats says how many floats)."""

    @staticmethod
    def forward(ctx, q, k, v, g, s0, scale, cu_seqlens):
        note_leaves(ctx, q.device)
        q, k, v, g = _rows(q), _rows(k), _rows(v), g.contiguous()
        s0 = None if s0 is None else s0.contiguous()
        dims = _shapes(q, k, v, g, s0, cu_seqlens)
        out, send, parts = _fwd(q, k, v, g, s0, cu_seqlens, dims, scale, True)
        ctx.save_for_backward(q, k, v, g, s0, cu_seqlens, send, parts)
        ctx.scale, ctx.dims = scale, dims
        ctx.set_materialize_grads(False)
        return out, send

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dsend):
        q, k, v, g, s0, cu, send, parts = ctx.saved_tensors
        dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else dout.contiguous()
        if dsend is not None:
            dsend = dsend.contiguous()
        grads = _bwd(q, k, v, g, s0, cu, ctx.dims, ctx.scale, send, parts, dout, dsend, ctx.needs_input_grad[4])
        return *grads, None, None


def linear_attention(q, k, v, g, s0=None, *, scale=None, cu_seqlens=None):
    """(out, send) of linear attention under autograd (shapes: linear_fwd). Without a
    gradient to keep anything for, calls of up to 12 tokens run token by token. A capture
    may hold this and its backward pass; see note_leaves for the one that is refused.
    Forward-mode and second derivatives are refused."""
    refuse_tangents("linear_attention", q, k, v, g, s0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, s0)):
        return LinearAttention.apply(q, k, v, g, s0, scale, cu_seqlens)
    if s0 is not None:
        s0 = s0.contiguous()
    return linear_fwd(q, k, v, g, s0, scale=scale, cu_seqlens=cu_seqlens)[:2]


def linear_step(q, k, v, g, s, *, scale=None, send=None):
    """One token of B sequences: q, k (B,Hk,K), v (B,H,V), g (B,H) or (H), s (B,H,K,V)
    -> out (B,H,V). ``s`` is updated in place, or left and the new state written to
    ``send``. No autograd."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, s, send)):
        raise RuntimeError("linear_step keeps nothing for a backward pass: call linear_attention, or use "
                           "torch.no_grad()")
    refuse_tangents("linear_step", q, k, v, g, s, send)
    q, k, v, g = _rows(q), _rows(k), _rows(v), g.contiguous()
    dims = _shapes(q, k, v, g, s, None, step=True)
    B, _, N, Hk, H, K, V = dims
    if send is None:
        send = s
    elif send is not s:
        _check_state(send, (N, H, K, V), "send")
        if send.device != q.device:
            raise ValueError("linear attention takes tensors of one GPU")
        if 0 < abs(send.data_ptr() - s.data_ptr()) < s.numel() * 4:
            raise ValueError("send must be s or lie apart from it")
    out = torch.empty(B, H, V, dtype=v.dtype, device=q.device)
    if B == 0:
        return out
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), s.data_ptr(), 0, qb, 0, qh, kb, 0, kh,
                      vb, 0, vh, *dims, DTYPES[q.dtype], g.dim() == 1,
                      K ** -0.5 if scale is None else float(scale), 0)
    rc = _native.on_device(q.device, _native.lib().snhip_op_linear_step_dev, args, out.data_ptr(), send.data_ptr())
    _native.check(rc, "snhip_op_linear_step_dev")
    torch.autograd.graph.increment_version(send)       # a graph that saved the old state refuses this one
    return out
