"""The embedding lookup on the GPU with its gradient: rows of a table by token ids, times
a factor (the model's lookup, sunnynet/model.py:60,93, has a factor of 1).

    y_i = scale table[id_i]        dtable[r] = scale (sum of dy_i over the i with id_i = r)

An id outside of the table (a padding of -1, say) gives a row of zeros and no gradient.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .delta import DTYPES, note_leaves, refuse_tangents

__all__ = ["Embed", "embed", "embed_bwd", "embed_fwd"]

MAX_R, MAX_D, MAX_N = 1 << 28, 1 << 20, (1 << 31) - 1


def _check(shape, dtype, device, ids):
    """(n, R, D) of a call, after its checks."""
    if len(shape) != 2 or not 1 <= shape[0] <= MAX_R or not 1 <= shape[1] <= MAX_D:
        raise ValueError(f"the table must be (R, D) with R from 1 to {MAX_R} and D from 1 to {MAX_D}")
    if dtype not in DTYPES:
        raise ValueError("the table must be float32, bfloat16 or float16")
    if ids.dtype != torch.int64 and ids.dtype != torch.int32 or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 or int64 tensor")
    if device.type != "cuda" or ids.device != device:
        raise ValueError("the embedding takes tensors of one GPU")
    n = ids.numel()
    if n > MAX_N:
        raise ValueError("fewer than 2^31 ids per call")
    return n, *shape


def embed_fwd(table, ids, scale=1.0):
    """table (R, D) contiguous float32, bfloat16 or float16, ids (...) contiguous int32 or
    int64 -> scale table[ids] (..., D) of the table's type. Without autograd."""
    n, R, D = _check(table.shape, table.dtype, table.device, ids)
    if not table.is_contiguous():
        raise ValueError("the table must be contiguous")
    y = torch.empty(*ids.shape, D, dtype=table.dtype, device=table.device)
    if n:
        rc = _native.on_device(table.device, _native.lib().snhip_op_embed_fwd_dev, table.data_ptr(), ids.data_ptr(),
                               ids.dtype == torch.int64, y.data_ptr(), n, R, D, scale, DTYPES[table.dtype])
        _native.check(rc, "snhip_op_embed_fwd_dev")
    return y


def embed_bwd(dy, ids, rows, scale=1.0):
    """The gradient of a table of ``rows`` rows: dy (..., D) contiguous -> (rows, D) of dy's
    type. Sums are float32, in the batch's order: the same call gives the same bits."""
    D = dy.shape[-1] if dy.dim() else 0
    if dy.shape[:-1] != ids.shape or not dy.is_contiguous():
        raise ValueError("dy must be contiguous, of the ids' shape and (D)")
    n, R, D = _check((rows, D), dy.dtype, dy.device, ids)
    if not n:
        return torch.zeros(R, D, dtype=dy.dtype, device=dy.device)
    L, kind = _native.lib(), DTYPES[dy.dtype]
    out = torch.empty(R, D, dtype=dy.dtype, device=dy.device)
    ws = torch.empty(L.snhip_op_embed_bwd_bytes(n, R, D, kind), dtype=torch.uint8, device=dy.device)
    rc = _native.on_device(dy.device, L.snhip_op_embed_bwd_dev, dy.data_ptr(), ids.data_ptr(), ids.dtype == torch.int64,
                           out.data_ptr(), ws.data_ptr(), n, R, D, scale, kind)
    _native.check(rc, "snhip_op_embed_bwd_dev")
    return out


class Embed(torch.autograd.Function):
    """The lookup under autograd; saves the ids."""

    @staticmethod
    def forward(ctx, table, ids, scale):
        note_leaves(ctx, table.device)
        ids = ids.contiguous()
        y = embed_fwd(table.contiguous(), ids, scale)
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return embed_bwd(dy.contiguous(), *ctx.saved_tensors, ctx.rows, ctx.scale), None, None


def embed(table, ids, scale=1.0):
    """scale table[ids] under autograd: table (R, D) float32, bfloat16 or float16, ids
    (...) int32 or int64 on the same GPU -> (..., D). Ids outside [0, R) give zeros. A
    capture may hold this and its backward pass; see note_leaves for the one that is
    refused. Forward-mode and second derivatives are refused."""
    refuse_tangents("embed", table)
    if table.requires_grad and torch.is_grad_enabled():
        return Embed.apply(table, ids, float(scale))
    return embed_fwd(table.contiguous(), ids.contiguous(), float(scale))
