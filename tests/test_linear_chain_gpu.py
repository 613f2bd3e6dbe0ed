"""The state of linear attention after many chunks: each chunk of fp32 and fp16 inputs is
added to it by one rounding, whatever the number of partial products that make it up.

Tolerance. A rounding to fp32 is off by at most half a step, rms over values of all sizes
0.42 2^-24 of the value. Without a decay the state grows as the root of the tokens, so n chunks
of 32, rounded independently, give 0.42 2^-24 sqrt(n / 2) of the state's rms. What a chunk adds
(weights, their products with v, sums over its tokens) is good to 2 2^-24 of its own rms, and
more so next to the state: 2^-24 (2 + 0.42 sqrt(n / 2)) in all. With a rounding for each of
the five or six partial products besides the decay's it would be 2^-24 (2 + 0.42 sqrt(6 n / 2))
at least.

A decay of a whole chunk, d = exp(sum of g), is fp32 itself and the same for all chunks here:
off by at most a step below 1, 2^-24, where exp(-32 2^-13) < d < 1. What was added j chunks
before the end is off by j times as much; with n like parts of random sign that makes
2^-24 sqrt(sum of j^2 / n) = 2^-24 n / sqrt(3) more. Without a decay d is 1, exactly.
"""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["fp32", "fp16"])
@pytest.mark.parametrize("decay", [0.0, 2.0 ** -13], ids=["none", "slow"])
def test_rounded_once_a_chunk(gpu, decay, dtype):
    B, T, H, D = 64, 4096, 8, 64           # as many blocks as fill the card: sequences in one part
    gen = torch.Generator(gpu).manual_seed(1)
    q, k = (torch.randn(B, T, 1, D, device=gpu, generator=gen).to(dtype) for _ in range(2))
    v = torch.randn(B, T, H, D, device=gpu, generator=gen).to(dtype)
    g = -decay * torch.rand(H, device=gpu, generator=gen)
    with torch.no_grad():
        _, send = runtime.linear_attention(q, k, v, g)
    n = T / 32
    room = 2.0 ** -24 * (2 + 0.42 * math.sqrt(n / 2) + (n / math.sqrt(3) if decay else 0))
    left = torch.arange(T - 1, -1, -1, device=gpu, dtype=torch.float64)
    for h in range(H):
        kw = k[:, :, 0].double() * torch.exp(left * g[h].double())[:, None]
        want = torch.matmul(kw.transpose(1, 2).contiguous(), v[:, :, h].double().contiguous())
        error = float((send[:, h].double() - want).square().mean().sqrt() / want.square().mean().sqrt())
        assert error <= room, f"head {h}: {error * 2 ** 24:.2f} of 2^-24"
