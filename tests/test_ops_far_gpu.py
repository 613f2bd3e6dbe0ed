"""The operators at the ends of their sizes: most heads, most sequences, widest values, and
arrays of more than 2^31 elements."""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta", "s0")


def inputs(B, T, Hk, H, K, V, dtype, seed):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    def unit(*s):
        x = rn(*s)
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-3)

    x = {"q": unit(B, T, Hk, K).to(dtype), "k": unit(B, T, Hk, K).to(dtype), "v": rn(B, T, H, V).to(dtype),
         "g": -torch.exp(rn(B, T, H) - 2), "beta": torch.sigmoid(2 * rn(B, T, H)), "s0": 0.3 * rn(B, H, K, V)}
    return [x[n] for n in NAMES]


def ref(q, k, v, g, beta, S):
    rep, outs = v.shape[2] // q.shape[2], []
    for t in range(q.shape[1]):
        qt, kt = (x[:, t].repeat_interleave(rep, 1) for x in (q, k))
        S = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (S * kt[..., None]).sum(2))
        S = S + kt[..., None] * u[:, :, None, :]
        outs.append((S * qt[..., None]).sum(2) * q.shape[-1] ** -0.5)
    return torch.stack(outs, 1), S


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 40, 1, 2, 128, 4096), (1, 34, 5, 65535, 1, 1), (65535, 14, 1, 1, 2, 3),
                                   (65535, 2, 1, 1, 4, 4)], ids=str)
def test_delta_at_its_largest(gpu, shape, dtype):
    """Against 64 bits. An fp32 sum of K + 64 terms, four products deep (and four times that for
    gradients): 4 (K + 64) 2^-24 of the largest value, and half a step of the type."""
    x = inputs(*shape, dtype, 1)
    x64 = [t.double().to(gpu).requires_grad_() for t in x]
    ro, rs = ref(*x64)
    gen = torch.Generator().manual_seed(2)
    do, ds = torch.randn(ro.shape, generator=gen).to(dtype).to(gpu), torch.randn(rs.shape, generator=gen).to(gpu)
    want = torch.autograd.grad((ro, rs), x64, (do.double(), ds.double()))
    leaf = [t.to(gpu).requires_grad_() for t in x]
    out, send = runtime.gated_delta(*leaf)
    got = torch.autograd.grad((out, send), leaf, (do, ds))
    with torch.no_grad():
        plain = runtime.gated_delta(*leaf)
    for n, a, b, grad in (("out", out, ro, 1), ("send", send, rs, 1), ("plain", plain[0], ro, 1), ("end", plain[1], rs, 1),
                          *(("d" + n, a, b, 4) for n, a, b in zip(NAMES, got, want))):
        tol = 4 * grad * (shape[4] + 64) * 2.0 ** -24 * b.abs().max() + torch.finfo(a.dtype).eps / 2 * b.abs()
        worst = float(((a.detach().double() - b.detach()).abs() - tol.detach()).max())
        assert worst <= 0, n


def test_delta_beyond_32_bits(gpu):
    """More than 2^31 values in v, out and their gradients. The state is forgotten at a chunk's
    first token near the end, so the tokens from there on have the bits of their own call."""
    T, H, K, V, at = 136000, 128, 128, 128, 136000 - 6 * 64
    assert T * H * V > 1 << 31
    gen = torch.Generator(gpu).manual_seed(3)
    bf = dict(dtype=torch.bfloat16, device=gpu)
    q, k = (torch.empty(1, T, 1, K, **bf).normal_(0, K ** -0.5, generator=gen) for _ in range(2))
    v, dout = (torch.empty(1, T, H, V, **bf).normal_(generator=gen) for _ in range(2))
    g, beta = (torch.rand(1, T, H, device=gpu, generator=gen) for _ in range(2))
    g = -0.2 * g
    g[:, at] = -math.inf

    def run(*leaf, dout):
        leaf = [t.requires_grad_() for t in leaf]
        out, send = runtime.gated_delta(*leaf)
        return out.detach(), send.detach(), *torch.autograd.grad((out, send), leaf, (dout, torch.ones_like(send)))

    whole = run(q, k, v, g, beta, dout=dout)
    tail = run(*(t.detach()[:, at:].clone() for t in (q, k, v, g, beta)), dout=dout[:, at:].clone())
    assert torch.equal(whole[1], tail[1])
    for a, b in zip((whole[0], *whole[2:]), (tail[0], *tail[2:])):
        assert torch.equal(a[:, at:], b)
    # and the first tokens have those of a call that ends with a chunk
    head = runtime.gated_delta(*(t.detach()[:, :640].clone() for t in (q, k, v, g, beta)))[0]
    assert torch.equal(whole[0][:, :640], head)


def test_norm_beyond_32_bits(gpu):
    R, D = (1 << 21) + 77, 1030
    gen = torch.Generator(gpu).manual_seed(4)
    x, dy = (torch.empty(R, D, dtype=torch.bfloat16, device=gpu).normal_(generator=gen) for _ in range(2))
    w = torch.rand(D, device=gpu, generator=gen)
    y, mean, rstd = runtime.norm_fwd(x, w, w, keep=True)
    dx, _, db = runtime.norm_bwd(dy, x, w, mean, rstd)
    part = slice(R - 300, R)
    own = runtime.norm_fwd(x[part], w, w, keep=True)
    assert all(torch.equal(a[part], b) for a, b in zip((y, mean, rstd), own))
    assert torch.equal(dx[part], runtime.norm_bwd(dy[part], x[part], w, *own[1:])[0])
    # 2^21 rows of random sign: partial sums of some 500 rows in a lane, then 272 of those
    want = torch.stack([dy[i:i + 100000].double().sum(0) for i in range(0, R, 100000)]).sum(0)
    size = torch.stack([dy[i:i + 100000].double().abs().sum(0) for i in range(0, R, 100000)]).sum(0)
    assert bool(((db.double() - want).abs() <= 800 * 2.0 ** -24 * size).all())


def test_sampling_beyond_32_bits(gpu):
    B, V = 2100, 1 << 20
    gen = torch.Generator(gpu).manual_seed(5)
    x = torch.empty(B, V, dtype=torch.bfloat16, device=gpu).normal_(0, 3, generator=gen)
    u = torch.rand(B, dtype=torch.float64, device=gpu, generator=gen)
    got = runtime.sample_tokens(x, u, 0.9, 300, 0.95)
    assert torch.equal(got[-50:], runtime.sample_tokens(x[-50:].clone(), u[-50:], 0.9, 300, 0.95))
    assert torch.equal(runtime.sample_tokens(x, u, 0.0)[-50:].long(), x[-50:].float().argmax(1))
