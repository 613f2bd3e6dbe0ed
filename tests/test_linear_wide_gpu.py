"""Linear attention's blocks of 128 columns, which calls of many tokens and heads take, against
its definition in 64 bits: all pairs of tokens at once. Tolerances as in test_linear_gpu.py."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime
from test_linear_gpu import BF16, F16, F32, NAMES, close, gradients_close, inputs

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
DECAYS = pytest.mark.parametrize("head_g", [False, True], ids=["token_g", "head_g"])


def pairs(q, k, v, g, s0):
    """The definition without its recurrence: every token with all before it."""
    B, T, Hk, K = q.shape
    H = v.shape[2]
    if not T:
        return v * 0, s0
    q, k = (x.repeat_interleave(H // Hk, 2).transpose(1, 2) for x in (q, k))
    v, c = v.transpose(1, 2), g.expand(B, T, H).cumsum(1).transpose(1, 2)
    gap = (c[..., :, None] - c[..., None, :]).masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -torch.inf)
    out = (gap.exp() * (q @ k.transpose(2, 3))) @ v + c.exp()[..., None] * (q @ s0)
    send = c[..., -1].exp()[..., None, None] * s0 + (k * (c[..., -1:] - c).exp()[..., None]).transpose(2, 3) @ v
    return K ** -0.5 * out.transpose(1, 2), send


def check(x, dtype, ref_of, cu=None):
    d = {n: t.double().cpu() for n, t in x.items()}
    want = ref_of(*(d[n] for n in NAMES))
    tol = 4 * (max(x["q"].shape[-1], x["v"].shape[-1]) + 64) * 2.0 ** -24
    with torch.no_grad():
        plain = runtime.linear_attention(*(x[n] for n in NAMES), cu_seqlens=cu)
    leaf = [x[n].clone().requires_grad_() for n in NAMES]
    out, send = runtime.linear_attention(*leaf, cu_seqlens=cu)
    for o, s in (plain, (out.detach(), send.detach())):
        close(o, want[0], dtype, tol, "out")
        close(s, want[1], F32, tol, "send")
    gen = torch.Generator().manual_seed(9)
    dout = torch.randn(out.shape, generator=gen).to(dtype).cuda()
    dsend = torch.randn(send.shape, generator=gen).cuda()
    got = torch.autograd.grad((out, send), leaf, (dout, dsend))
    gradients_close(x, got, dout, dsend, ref_of)


SHAPES = [  # B, T, Hk, H, K, V: in parts and, the second, in none; the state by 128 x 128, 64 x 128 and 128 x 64
    (2, 520, 8, 16, 128, 128), (32, 40, 16, 16, 128, 128), (1, 1100, 4, 8, 100, 130), (3, 700, 8, 8, 72, 128),
    (4, 520, 8, 8, 128, 40), (4, 520, 8, 8, 33, 100),
]


@TYPES
@DECAYS
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(gpu, shape, head_g, dtype):
    B, T, Hk, H, K, V = shape
    assert B * T * H * -(-V // 128) >= 256 * 64            # fewer take blocks of 64 columns
    check(inputs(*shape, dtype, seed=sum(shape), head_g=head_g), dtype, pairs)


@TYPES
@DECAYS
def test_packed(gpu, head_g, dtype):
    edges = [0, 700, 700, 701, 2090]
    T, Hk, H, K, V = 2100, 4, 8, 128, 128
    spans = list(zip(edges, edges[1:]))
    x = inputs(1, T, Hk, H, K, V, dtype, seed=7, N=len(spans), head_g=head_g)

    def packed(q, k, v, g, s0):
        res = [pairs(q[:, a:e], k[:, a:e], v[:, a:e], g if g.dim() == 1 else g[:, a:e], s0[i:i + 1])
               for i, (a, e) in enumerate(spans)]
        return torch.cat([r[0] for r in res] + [v[:, edges[-1]:] * 0], 1), torch.cat([r[1] for r in res])

    check(x, dtype, packed, torch.tensor(edges, dtype=torch.int32, device="cuda"))
