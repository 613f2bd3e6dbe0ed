"""The common norm of many gradients on the GPU, and their clipping by it, without a host
synchronization and without copies: the tensors' addresses travel with the launches.

    norm = sqrt(sum of all x^2)        x <- x min(1, max_norm / (norm + 1e-6))
"""
from __future__ import annotations

import struct
from array import array
from operator import attrgetter

import torch

from .. import _native
from .delta import DTYPES, refuse_tangents

__all__ = ["clip_grad_norm", "grad_norm"]

MAX_TENSORS, MAX_ELEMENTS = 1 << 20, 1 << 36
_ARGS = struct.Struct("4Pqd1P")        # SnHipClip
_dtype = attrgetter("dtype")


def _addresses(tensors, what):
    """(addresses, sizes, kinds, device index) of a list of tensors, after its checks."""
    try:
        where = set(map(torch.Tensor.get_device, tensors))
    except TypeError:
        raise ValueError("the gradients must be tensors: leave out parameters without one") from None
    if len(where) > 1 or -1 in where:
        raise ValueError(f"{what} must be tensors of one GPU")
    dtypes = set(map(_dtype, tensors))
    if not dtypes <= DTYPES.keys():
        raise ValueError(f"{what} must be float32, bfloat16 or float16")
    if len(dtypes) == 1:
        kinds = array("i", [DTYPES[dtypes.pop()]]) * len(tensors)
    else:
        kinds = array("i", [DTYPES[d] for d in map(_dtype, tensors)])
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise ValueError(f"{what} must be contiguous")
    sizes = array("q", [*map(torch.Tensor.numel, tensors)])
    return array("Q", [*map(torch.Tensor.data_ptr, tensors)]), sizes, kinds, where.pop() if where else None


def _run(tensors, max_norm, out):
    if len(tensors) >= MAX_TENSORS:
        raise ValueError(f"fewer than {MAX_TENSORS} tensors per call")
    x, sizes, kinds, at = _addresses(tensors, "the gradients")
    if at is None:
        raise ValueError("no gradients")
    if max(sizes) >= MAX_ELEMENTS:
        raise ValueError(f"fewer than {MAX_ELEMENTS} elements per tensor")
    y = x
    if out is not tensors and out is not None:
        if len(out) != len(tensors):
            raise ValueError("out must hold a tensor for each gradient")
        y, out_sizes, out_kinds, out_at = _addresses(out, "out")
        if out_sizes != sizes or out_kinds != kinds or out_at != at:
            raise ValueError("out must hold tensors like the gradients")
    device = torch.device("cuda", at)
    L = _native.lib()
    norm = torch.empty((), dtype=torch.float32, device=device)
    ws = torch.empty(L.snhip_op_clip_doubles(len(tensors)), dtype=torch.float64, device=device)
    args = _ARGS.pack(x.buffer_info()[0], 0 if out is None else y.buffer_info()[0], sizes.buffer_info()[0],
                      kinds.buffer_info()[0], len(tensors), max_norm, ws.data_ptr())
    rc = _native.on_device(device, L.snhip_op_clip_dev, args, norm.data_ptr())
    if rc == -1:
        raise ValueError("out must lie apart from the gradients (or be them), and no two gradients may share memory")
    _native.check(rc, "snhip_op_clip_dev")
    return norm


def grad_norm(grads):
    """The norm of all elements of the gradients (contiguous float32, bfloat16 or float16
    tensors of one GPU, each of its own type) -> float32 scalar on the device. Squares are
    summed in 64 bits in a fixed order: the same calls give the same bits. Not
    differentiable; forward-mode derivatives are refused."""
    grads = list(grads)
    refuse_tangents("grad_norm", *grads)
    return _run(grads, 0.0, None)


@torch.no_grad()
def clip_grad_norm(grads, max_norm, *, out=None):
    """Multiplies the gradients (see grad_norm) by min(1, max_norm / (norm + 1e-6)), in
    place, or into the tensors of ``out`` (like the gradients), and returns the norm before,
    a float32 scalar on the device. Where nothing is to clip, gradients in place are not
    touched. A norm that is infinite (some value is) makes finite values 0, one that is NaN
    makes all NaN. An infinite ``max_norm`` clips nothing. Two gradients that share memory
    are refused. Not differentiable; forward-mode derivatives are refused."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    grads = list(grads)
    if out is not None:
        out = list(out)
    refuse_tangents("clip_grad_norm", *grads, *(out or ()))
    if any(t is not None and t.requires_grad and t.is_leaf for t in (grads if out is None else out)):
        raise RuntimeError("a leaf that requires a gradient cannot be written in place")
    norm = _run(grads, max_norm, grads if out is None else out)
    torch.autograd.graph.increment_version(grads if out is None else out)      # a graph that saved one refuses it
    return norm
