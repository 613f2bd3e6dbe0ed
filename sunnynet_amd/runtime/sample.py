"""The next token of every row of a batch of logits, chosen on the GPU from given
random numbers, with the scheduler's rules (sunnynet/serve.py:29-56): temperature,
then top-k, top-p and min-p, then the inverse of the remaining distribution in index
order.
"""
from __future__ import annotations

import struct

import torch

from .. import _native
from .delta import DTYPES

__all__ = ["sample_tokens"]

MAX_V = 1 << 20
_ARGS = struct.Struct("6P3d5q")        # SnHipSample


def _setting(x, name, B, device, dtype):
    """(tensor or None, value) of a per-row or common setting."""
    if not torch.is_tensor(x):
        return None, x
    if x.shape != (B,) or x.device != device or x.dtype.is_complex or x.dtype == torch.bool:
        raise ValueError(f"{name} must be a number or a vector of one number per row on the logits' device")
    if dtype == torch.int32 and x.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
        # to what filters alike, so that 32 bits do not make another number of it
        x = (x.double().nan_to_num(0) if x.is_floating_point() else x.to(torch.int64)).clamp(0, MAX_V)
    return x.to(dtype).contiguous(), 0


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, drew=False):
    """logits (B, V) float32, bfloat16 or float16 (rows contiguous, any row stride), u (B)
    float64 or float32 in [0, 1) -> tokens (B) int32 on the device, without a host
    synchronization. Each setting is one number or a vector of B. Per row:

    * temperature <= 0: the first maximal logit (a NaN counts as maximal);
    * else z = logit / temperature in 64 bits, weight exp(z - max z), and
      top_k in [1, V) keeps the k largest z (and all equal to the k-th);
    * top_p in (0, 1) keeps, in descending order (equal ones by index), the tokens
      before which the kept share is at most top_p;
    * min_p keeps weights of at least min_p (the largest weight is 1);
    * the token is the first whose running share of what is kept exceeds u.

    A row whose weights have no finite positive sum gives its first maximal logit. With
    ``drew`` the result is (2, B): the tokens, and 1 where u chose the row's token, else 0."""
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= MAX_V:
        raise ValueError(f"logits must be (B, V) with V from 1 to {MAX_V}")
    B, V = logits.shape
    if logits.dtype not in DTYPES:
        raise ValueError("logits must be float32, bfloat16 or float16")
    if not logits.is_cuda:
        raise ValueError("sample_tokens takes device tensors")
    if not torch.is_tensor(u) or u.shape != (B,) or u.dtype not in (torch.float32, torch.float64) \
            or u.device != logits.device:
        raise ValueError("u must be a float32 or float64 vector of one number per row on the logits' device")
    if V > 1 and logits.stride(1) != 1 or B > 1 and logits.stride(0) < 0:
        logits = logits.contiguous()
    dev = logits.device
    tokens = torch.empty((2, B) if drew else B, dtype=torch.int32, device=dev)
    if B == 0:
        return tokens
    f64 = torch.float64
    u = u.to(f64).contiguous()
    t, t0 = _setting(temperature, "temperature", B, dev, f64)
    k, k0 = _setting(top_k, "top_k", B, dev, torch.int32)
    p, p0 = _setting(top_p, "top_p", B, dev, f64)
    m, m0 = _setting(min_p, "min_p", B, dev, f64)
    args = _ARGS.pack(logits.data_ptr(), u.data_ptr(), *(0 if x is None else x.data_ptr() for x in (t, k, p, m)),
                      float(t0), float(p0), float(m0), min(max(int(k0), 0), MAX_V), B, V, logits.stride(0), DTYPES[logits.dtype])
    rc = _native.on_device(dev, _native.lib().snhip_op_sample_drew_dev, args, tokens.data_ptr(),
                           tokens[1].data_ptr() if drew else None)
    _native.check(rc, "snhip_op_sample_drew_dev")
    return tokens
