"""The gated delta rule on the GPU: a matrix state per head with decay and an
error-correcting write, as prompts and training run it (chunked) and token by
token. No counterpart in the reference.

Per sequence and value head, with ``a = exp(g)``:

    u_t = beta_t (v_t - a_t S_{t-1}^T k_t)
    S_t = a_t S_{t-1} + k_t u_t^T
    out_t = scale S_t^T q_t

Value head ``h`` of ``H`` reads query and key head ``h // (H // Hk)``. States and
sums are fp32 whatever the inputs' type. ``g <= 0`` is meant; ``-inf`` forgets the
state exactly. A value that is not finite makes its sequence and head NaN from the
chunk of 32 tokens that holds it on.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native

__all__ = ["GatedDelta", "delta_bwd", "delta_fwd", "delta_step", "gated_delta"]

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_K, MAX_V, MAX_HEADS, MAX_STRIDE = 128, 4096, 65535, 1 << 24
STEP_TOKENS = 12               # at most this many tokens run token by token
_ARGS = struct.Struct("7P9q8qd2P")     # SnHipDelta
_GRAD = struct.Struct("9P")            # SnHipDeltaGrad


def note_leaves(ctx, device):
    """Torch makes a leaf's gradient node on the stream that first uses the leaf, keeps it
    while a graph of it lives, and waits on that stream in every backward pass through it.
    Inside a capture no wait on the default stream is possible, and the process ends at it:
    nodes that are seen on the default stream are marked, and a capture that meets a marked
    one is refused."""
    if device.type != "cuda":
        return                 # refused later
    on_default = not _native.raw_stream(device)        # which cannot be captured
    if not on_default and not torch.cuda.is_current_stream_capturing():
        return
    for node, _ in ctx.next_functions:
        if node is None or node.name() != "torch::autograd::AccumulateGrad":
            continue
        if on_default:
            node.metadata["snhip_default_stream"] = True
        elif "snhip_default_stream" in node.metadata:
            raise RuntimeError("a graph of these leaves, made on the default stream, is still alive: delete its "
                               "outputs before capturing, or make it on another stream")


def refuse_tangents(name, *tensors):
    """Forward-mode derivatives are not there, and a result without one would count as
    constant. Dual tensors need no requires_grad, and carry their tangents under no_grad.
    There are none outside of a dual level (asked first: 2 us a call less, where this torch
    tells it)."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _shapes(q, k, v, g, beta, s0, cu, step=False):
    """(B, T, N, Hk, H, K, V) of a call, after its checks. step: one token, without T axes."""
    if step:
        (B, Hk, K), T = q.shape, 1
        H, V = v.shape[1:]
        if k.shape != q.shape or v.shape[0] != B or g.shape != (B, H) or beta.shape != (B, H):
            raise ValueError("shape mismatch: q, k (B,Hk,K); v (B,H,V); g, beta (B,H)")
    else:
        if q.dim() != 4 or v.dim() != 4 or k.shape != q.shape:
            raise ValueError("shape mismatch: q, k (B,T,Hk,K); v (B,T,H,V)")
        B, T, Hk, K = q.shape
        H, V = v.shape[2:]
        if v.shape[:2] != (B, T) or g.shape != (B, T, H) or beta.shape != (B, T, H):
            raise ValueError("shape mismatch: q, k (B,T,Hk,K); v (B,T,H,V); g, beta (B,T,H)")
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{H} value heads cannot share {Hk} query and key heads evenly")
    if not 1 <= K <= MAX_K or not 1 <= V <= MAX_V or H > MAX_HEADS:
        raise ValueError(f"head sizes up to K = {MAX_K}, V = {MAX_V} and up to {MAX_HEADS} heads: "
                         f"got K = {K}, V = {V}, {H} heads")
    if H * max(K, V) >= MAX_STRIDE:
        raise ValueError(f"H * K and H * V must be below {MAX_STRIDE}")
    if B * T >= 1 << 30:
        raise ValueError("B * T must be below 2^30")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be float32, bfloat16 or float16, all three the same")
    if g.dtype != torch.float32 or beta.dtype != torch.float32:
        raise ValueError("g and beta must be float32")
    N = B
    if cu is not None:
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 2 or not cu.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous int32 vector of at least two edges")
        if B != 1:
            raise ValueError("with cu_seqlens the sequences lie end to end in one batch entry: B must be 1")
        N = cu.shape[0] - 1
    if N > 65535:
        raise ValueError("at most 65535 sequences per call")
    if not step and (B * -(-T // 32) if cu is None else T // 32 + N) >= 1 << 23:
        raise ValueError("fewer than 2^23 chunks of 32 tokens per call")
    if s0 is not None:
        _check_state(s0, (N, H, K, V), "s0")
    dev = q.device
    if not q.is_cuda or k.device != dev or v.device != dev or g.device != dev or beta.device != dev \
            or s0 is not None and s0.device != dev or cu is not None and cu.device != dev:
        raise ValueError("the delta rule takes tensors of one GPU")
    return B, T, N, Hk, H, K, V


def _check_state(s, shape, name):
    if s.shape != shape or s.dtype != torch.float32 or not s.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {tuple(shape)}")


def _rows(t):
    """t with its last axis contiguous; the others may have any stride below MAX_STRIDE."""
    if (t.stride(-1) == 1 or t.shape[-1] == 1) and (t.dim() < 4 or t.stride(1) < MAX_STRIDE):
        return t
    return t.contiguous()


def _pack(q, k, v, g, beta, s0, cu, dims, scale, chunks=None, states=None):
    return _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), _ptr(s0), _ptr(cu),
                      *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *dims, DTYPES[q.dtype], scale,
                      _ptr(chunks), _ptr(states))


def delta_fwd(q, k, v, g, beta, s0=None, *, scale=None, cu_seqlens=None, keep=False):
    """q, k (B,T,Hk,K), v (B,T,H,V), g, beta (B,T,H), s0 (B,H,K,V) or None ->
    (out (B,T,H,V), send (B,H,K,V), saved), without autograd. The last axes of q, k and
    v are contiguous or copied; their other strides are free. With ``cu_seqlens`` (N + 1
    int32 edges on the device, not decreasing) B is 1, sequence n holds tokens
    ``[cu[n], cu[n+1])``, s0 and send are (N,H,K,V), and tokens of no sequence give 0.
    ``saved``: what delta_bwd needs (``keep``), else None. ``scale``: K ** -0.5 if None."""
    q, k, v, g, beta = _rows(q), _rows(k), _rows(v), g.contiguous(), beta.contiguous()
    dims = _shapes(q, k, v, g, beta, s0, cu_seqlens)
    return _fwd(q, k, v, g, beta, s0, cu_seqlens, dims, scale, keep)


def _fwd(q, k, v, g, beta, s0, cu_seqlens, dims, scale, keep):
    B, T, N, Hk, H, K, V = dims
    scale = K ** -0.5 if scale is None else float(scale)
    new = torch.empty if cu_seqlens is None else torch.zeros
    out = new(B, T, H, V, dtype=v.dtype, device=q.device)
    send = torch.empty(N, H, K, V, dtype=torch.float32, device=q.device)
    if B * T == 0 or N == 0:
        send.zero_() if s0 is None else send.copy_(s0)
        return out, send, (None, None) if keep else None
    L = _native.lib()
    chunks = states = None
    if keep or cu_seqlens is not None or T > STEP_TOKENS:
        sizes = _pack(q, k, v, g, beta, s0, cu_seqlens, dims, scale)
        chunks = torch.empty(L.snhip_op_delta_chunk_floats(sizes), dtype=torch.float32, device=q.device)
        if keep:
            states = torch.empty(L.snhip_op_delta_state_floats(sizes), dtype=torch.float32, device=q.device)
    rc = _native.on_device(q.device, L.snhip_op_delta_fwd_dev,
                           _pack(q, k, v, g, beta, s0, cu_seqlens, dims, scale, chunks, states), out.data_ptr(),
                           send.data_ptr())
    _native.check(rc, "snhip_op_delta_fwd_dev")
    return out, send, (chunks, states) if keep else None


def delta_bwd(q, k, v, g, beta, s0, saved, dout, dsend=None, *, scale=None, cu_seqlens=None, need_ds0=True):
    """Gradients of delta_fwd(..., keep=True) -> (dq, dk, dv, dg, dbeta, ds0): dout
    (B,T,H,V) of the inputs' type, dsend (N,H,K,V) float32 or None (zeros); ds0 is
    None unless ``need_ds0``. The same calls give the same bits."""
    q, k, v, g, beta = _rows(q), _rows(k), _rows(v), g.contiguous(), beta.contiguous()
    dims = _shapes(q, k, v, g, beta, s0, cu_seqlens)
    B, T, N, Hk, H, K, V = dims
    if dout.shape != (B, T, H, V) or dout.dtype != v.dtype or dout.device != q.device:
        raise ValueError("dout must be (B,T,H,V), of the inputs' type and device")
    if dsend is not None:
        _check_state(dsend, (N, H, K, V), "dsend")
        if dsend.device != q.device:
            raise ValueError("the delta rule takes tensors of one GPU")
    if B * T and N:
        L, sizes = _native.lib(), _pack(q, k, v, g, beta, s0, cu_seqlens, dims, 1.0)
        sizes = L.snhip_op_delta_chunk_floats(sizes), L.snhip_op_delta_state_floats(sizes)
        if not saved or any(t is None or t.shape != (n,) or t.dtype != torch.float32 or t.device != q.device
                            or not t.is_contiguous() for t, n in zip(saved, sizes)):
            raise ValueError("saved must be delta_fwd's, of the same shapes, with keep=True")
    return _bwd(q, k, v, g, beta, s0, cu_seqlens, dims, scale, saved, dout.contiguous(), dsend, need_ds0)


def _bwd(q, k, v, g, beta, s0, cu_seqlens, dims, scale, saved, dout, dsend, need_ds0):
    B, T, N, Hk, H, K, V = dims
    scale = K ** -0.5 if scale is None else float(scale)
    new = torch.empty if cu_seqlens is None else torch.zeros
    dq, dk = (new(B, T, Hk, K, dtype=q.dtype, device=q.device) for _ in range(2))
    dv = new(B, T, H, V, dtype=q.dtype, device=q.device)
    dg, db = (new(B, T, H, dtype=torch.float32, device=q.device) for _ in range(2))
    ds0 = torch.empty(N, H, K, V, dtype=torch.float32, device=q.device) if need_ds0 else None
    if B * T == 0 or N == 0:
        if need_ds0:
            ds0.zero_() if dsend is None else ds0.copy_(dsend)
        return dq, dk, dv, dg, db, ds0
    L = _native.lib()
    chunks, states = saved
    args = _pack(q, k, v, g, beta, s0, cu_seqlens, dims, scale, chunks, states)
    ws = torch.empty(L.snhip_op_delta_bwd_floats(args), dtype=torch.float32, device=q.device)
    grads = _GRAD.pack(dout.data_ptr(), _ptr(dsend), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
                       db.data_ptr(), _ptr(ds0), ws.data_ptr())
    rc = _native.on_device(q.device, L.snhip_op_delta_bwd_dev, args, grads)
    _native.check(rc, "snhip_op_delta_bwd_dev")
    return dq, dk, dv, dg, db, ds0


class GatedDelta(torch.autograd.Function):
    """The gated delta rule under autograd: (out, send) of delta_fwd, gradients of
    delta_bwd. Keeps the forward's two workspaces, in fp32 per head: a state (K to 64 or
    128, V to a multiple of 16) for every 32 tokens (64 in 16 bits with K > 64), V errors
    a token and 99 floats a token of chunk matrices; a long sequence of few heads also its
    parts' maps (snhip_op_delta_chunk_floats and snhip_op_delta_state_floats say how many)."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, s0, scale, cu_seqlens):
        note_leaves(ctx, q.device)
        q, k, v, g, beta = _rows(q), _rows(k), _rows(v), g.contiguous(), beta.contiguous()
        s0 = None if s0 is None else s0.contiguous()
        dims = _shapes(q, k, v, g, beta, s0, cu_seqlens)
        out, send, saved = _fwd(q, k, v, g, beta, s0, cu_seqlens, dims, scale, True)
        ctx.save_for_backward(q, k, v, g, beta, s0, cu_seqlens, *saved)
        ctx.scale, ctx.dims = scale, dims
        ctx.set_materialize_grads(False)
        return out, send

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dsend):
        q, k, v, g, beta, s0, cu, *saved = ctx.saved_tensors
        dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else dout.contiguous()
        if dsend is not None:
            dsend = dsend.contiguous()
        grads = _bwd(q, k, v, g, beta, s0, cu, ctx.dims, ctx.scale, saved, dout, dsend, ctx.needs_input_grad[5])
        return *grads, None, None


def gated_delta(q, k, v, g, beta, s0=None, *, scale=None, cu_seqlens=None):
    """(out, send) of the gated delta rule under autograd (shapes: delta_fwd). Without
    a gradient to keep anything for, calls of up to 12 tokens run token by token. A capture
    may hold this and its backward pass; see note_leaves for the one that is refused.
    Forward-mode and second derivatives are refused."""
    refuse_tangents("gated_delta", q, k, v, g, beta, s0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, s0)):
        return GatedDelta.apply(q, k, v, g, beta, s0, scale, cu_seqlens)
    if s0 is not None:
        s0 = s0.contiguous()
    return delta_fwd(q, k, v, g, beta, s0, scale=scale, cu_seqlens=cu_seqlens)[:2]


def delta_step(q, k, v, g, beta, s, *, scale=None, send=None):
    """One token of B sequences: q, k (B,Hk,K), v (B,H,V), g, beta (B,H), s (B,H,K,V)
    -> out (B,H,V). ``s`` is updated in place, or left and the new state written to
    ``send``. No autograd."""
    if q.dim() != 3 or v.dim() != 3 or k.dim() != 3 or g.dim() != 2 or beta.dim() != 2:
        raise ValueError("shape mismatch: q, k (B,Hk,K); v (B,H,V); g, beta (B,H)")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or s.requires_grad
                                    or send is not None and send.requires_grad):
        raise RuntimeError("delta_step keeps nothing for a backward pass: call gated_delta, or use torch.no_grad()")
    refuse_tangents("delta_step", q, k, v, g, beta, s, send)
    q, k, v, g, beta = _rows(q), _rows(k), _rows(v), g.contiguous(), beta.contiguous()
    dims = _shapes(q, k, v, g, beta, s, None, step=True)
    B, _, N, Hk, H, K, V = dims
    if send is None:
        send = s
    elif send is not s:
        _check_state(send, (N, H, K, V), "send")
        if send.device != q.device:
            raise ValueError("the delta rule takes tensors of one GPU")
        if 0 < abs(send.data_ptr() - s.data_ptr()) < s.numel() * 4:
            raise ValueError("send must be s or lie apart from it")
    out = torch.empty(B, H, V, dtype=v.dtype, device=q.device)
    if B == 0:
        return out
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), s.data_ptr(), 0,
                      qb, 0, qh, kb, 0, kh, vb, 0, vh, *dims, DTYPES[q.dtype],
                      K ** -0.5 if scale is None else float(scale), 0, 0)
    rc = _native.on_device(q.device, _native.lib().snhip_op_delta_step_dev, args, out.data_ptr(), send.data_ptr())
    _native.check(rc, "snhip_op_delta_step_dev")
    torch.autograd.graph.increment_version(send)       # a graph that saved the old state refuses this one
    return out
