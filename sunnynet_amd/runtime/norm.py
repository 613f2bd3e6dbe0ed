"""Layer norm on the GPU with its gradients, for training beside the fused block
core and for serving. The formula is the model's (sunnynet/ops.py:38-47): centred,
divided by ``sqrt(var + eps)``, times a gain, plus a centre.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .delta import DTYPES, _ptr, note_leaves, refuse_tangents

__all__ = ["LayerNorm", "layer_norm", "norm_bwd", "norm_fwd"]

MAX_D = 16384


def _check(x, w, b):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_D:
        raise ValueError(f"x must be (..., D) with D from 1 to {MAX_D}")
    if x.dtype not in DTYPES or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32, bfloat16 or float16 tensor")
    D = x.shape[-1]
    for t in (w, b):
        if t is not None and (t.shape != (D,) or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError("weight and bias must be contiguous float32 vectors of length D")
    if not x.is_cuda or any(t is not None and t.device != x.device for t in (w, b)):
        raise ValueError("layer norm takes tensors of one GPU")
    R = x.numel() // D
    if R >= 1 << 31:
        raise ValueError("fewer than 2^31 rows per call")
    return R, D


def norm_fwd(x, weight=None, bias=None, eps=1e-5, *, keep=False):
    """x (..., D) -> (y, mean, rstd): y of x's type; the row statistics in float32
    with ``keep``, else None. weight, bias: (D) float32 or None. Without autograd."""
    R, D = _check(x, weight, bias)
    y = torch.empty_like(x)
    mean, rstd = (torch.empty(R, dtype=torch.float32, device=x.device) for _ in range(2)) if keep else (None, None)
    if R:
        rc = _native.on_device(x.device, _native.lib().snhip_op_norm_fwd_dev, x.data_ptr(), _ptr(weight), _ptr(bias),
                               y.data_ptr(), _ptr(mean), _ptr(rstd), R, D, eps, DTYPES[x.dtype])
        _native.check(rc, "snhip_op_norm_fwd_dev")
    return y, mean, rstd


def norm_bwd(dy, x, weight, mean, rstd, *, need=(True, True, True)):
    """Gradients of norm_fwd(..., keep=True) -> (dx, dweight, dbias), each None where
    ``need`` says so. The sums over rows run in a fixed order."""
    R, D = _check(x, weight, None)
    if any(t is None for t in (mean, rstd)):
        raise ValueError("mean and rstd must be norm_fwd's")
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device or not dy.is_contiguous():
        raise ValueError("dy must be contiguous and like x")
    if any(t.shape != (R,) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous()
           for t in (mean, rstd)):
        raise ValueError("mean and rstd must be norm_fwd's")
    return _bwd(dy, x, weight, mean, rstd, need, R, D)


def _bwd(dy, x, weight, mean, rstd, need, R, D):
    L = _native.lib()
    dx = torch.empty_like(x) if need[0] else None
    new = torch.empty if R else torch.zeros
    dw, db = (new(D, dtype=torch.float32, device=x.device) if n else None for n in need[1:])
    if R and any(need):
        ws = None
        if need[1] or need[2]:
            ws = torch.empty(L.snhip_op_norm_bwd_floats(R, D), dtype=torch.float32, device=x.device)
        rc = _native.on_device(x.device, L.snhip_op_norm_bwd_dev, dy.data_ptr(), x.data_ptr(), _ptr(weight),
                               mean.data_ptr(), rstd.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), R, D,
                               DTYPES[x.dtype])
        _native.check(rc, "snhip_op_norm_bwd_dev")
    return dx, dw, db


class LayerNorm(torch.autograd.Function):
    """Layer norm under autograd; saves x and two floats per row."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        note_leaves(ctx, x.device)
        x = x.contiguous()
        weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
        y, mean, rstd = norm_fwd(x, weight, bias, eps, keep=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        return *_bwd(dy.contiguous(), x, weight, mean, rstd, ctx.needs_input_grad[:3], mean.shape[0], x.shape[-1]), None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, under
    autograd: x (..., D) float32, bfloat16 or float16, weight and bias (D) float32 or
    None. Statistics and sums are float32. A capture may hold this and its backward pass;
    see note_leaves for the one that is refused. Forward-mode and second derivatives are
    refused."""
    refuse_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return LayerNorm.apply(x, weight, bias, float(eps))
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    return norm_fwd(x.contiguous(), weight, bias, float(eps))[0]
