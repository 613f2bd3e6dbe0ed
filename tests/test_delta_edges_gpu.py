"""The gated delta rule where its workspaces, its operands' bits or its packed sequences
end. The 64-bit definition goes token by token, as the operator states it."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta", "s0")


def inputs(B, T, Hk, H, K, V, dtype, seed, N=None):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    def unit(*s):
        x = rn(*s)
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-3)

    x = {"q": unit(B, T, Hk, K).to(dtype), "k": unit(B, T, Hk, K).to(dtype), "v": rn(B, T, H, V).to(dtype),
         "g": -torch.exp(rn(B, T, H) - 2), "beta": torch.sigmoid(2 * rn(B, T, H)),
         "s0": 0.3 * rn(B if N is None else N, H, K, V)}
    return {n: t.cuda() for n, t in x.items()}


def test_records_that_fill_their_pages(gpu):
    """512 chunks of 32 heads: their records fill whole pages of 2 MB, so nothing lies behind
    the last one. Batch entries have the bits of their own calls."""
    x = inputs(8, 2048, 1, 32, 8, 16, torch.float32, 50)
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf)
    gen = torch.Generator().manual_seed(51)
    do, ds = torch.randn(out.shape, generator=gen).cuda(), torch.randn(send.shape, generator=gen).cuda()
    got = torch.autograd.grad((out, send), leaf, (do, ds))
    for b in (0, 7):
        one = [t.detach()[b:b + 1].clone().requires_grad_() for t in leaf]
        o, s = runtime.gated_delta(*one)
        assert torch.equal(o[0], out[b]) and torch.equal(s[0], send[b])
        for a, g in zip(torch.autograd.grad((o, s), one, (do[b:b + 1], ds[b:b + 1])), got):
            assert torch.equal(a[0], g[b])
