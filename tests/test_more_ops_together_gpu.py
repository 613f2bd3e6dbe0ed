"""A recurrent language model of one block as a training step and a server use the
operators: embedding, layer norm, linear attention, their gradients through plain torch
layers, clipping; against the same model in 64 bits, in a captured training step, and served
token by token.

Tolerances, fixed before the first run. The model's matrices are fp32 torch products of at
most 96 terms, the operators hold fp32; a gradient passes about ten such stages, each off by
at most some 100 2^-24 = 6e-6 of the sizes involved: 1e-4 of the largest entry. Clipping
multiplies by a factor that is as far off as the norm: 1e-4 more.
"""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime
from test_linear_gpu import ref

pytestmark = pytest.mark.gpu
D, Hk, H, K, V, VOCAB = 48, 2, 4, 16, 24, 97


def weights(seed=0):
    g = torch.Generator().manual_seed(seed)

    def rn(*s, std=0.2):
        return std * torch.randn(*s, generator=g)

    return {"embed": rn(VOCAB, D), "w1": 1 + rn(D), "b1": rn(D), "qk": rn(2 * Hk * K, D), "v": rn(H * V, D),
            "g": rn(H), "out": rn(D, H * V), "w2": 1 + rn(D), "b2": rn(D)}


def embed64(table, ids, scale):
    return torch.where((ids >= 0)[..., None], table[ids.clamp(min=0)] * scale, 0.0)


def norm64(x, w, b, eps):
    d = x - x.mean(-1, keepdim=True)
    return d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * w + b


def model(p, tokens, s0, embed, norm, mix):
    """tokens (B, T) -> logits (B, T, VOCAB), state."""
    B, T = tokens.shape
    x = embed(p["embed"], tokens, math.sqrt(D))
    h = norm(x, p["w1"], p["b1"], 4.1e-4)
    q, k = (h @ p["qk"].t()).view(B, T, 2, Hk, K).unbind(2)
    v = (h @ p["v"].t()).view(B, T, H, V)
    o, s = mix(q, 0.2 * k, v, -torch.exp(p["g"] - 1.0), s0)
    x = x + o.reshape(B, T, H * V) @ p["out"].t()
    return norm(x, p["w2"], p["b2"], 4.1e-4) @ p["embed"].t(), s


def loss_of(logits, targets):
    z = logits - logits.logsumexp(-1, keepdim=True)
    return -(z.gather(-1, targets.clamp(min=0)[..., None])[..., 0] * (targets >= 0)).sum() / (targets >= 0).sum()


OWN = runtime.embed, runtime.layer_norm, runtime.linear_attention


def batch(seed, B=3, T=150):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, VOCAB, (B, T + 1), generator=g)
    tokens[1, 100:] = -1                    # a shorter row, padded
    return tokens, 0.1 * torch.randn(B, H, K, V, generator=g)


def test_trained(gpu):
    p = weights()
    tokens, s0 = batch(1)
    p64 = {n: t.double().requires_grad_() for n, t in p.items()}
    lg, s = model(p64, tokens[:, :-1], s0.double(), embed64, norm64, ref)
    want = torch.autograd.grad(loss_of(lg, tokens[:, 1:]) + s.square().mean(), list(p64.values()))
    pd, td = {n: t.cuda().requires_grad_() for n, t in p.items()}, tokens.cuda()
    out, sd = model(pd, td[:, :-1], s0.cuda(), *OWN)
    got = torch.autograd.grad(loss_of(out, td[:, 1:]) + sd.square().mean(), list(pd.values()))
    assert (out.double().cpu() - lg).abs().max() <= 1e-4 * lg.abs().max()
    assert (sd.double().cpu() - s).abs().max() <= 1e-4 * s.abs().max()
    for n, a, b in zip(p, got, want):
        assert (a.double().cpu() - b).abs().max() <= 1e-4 * b.abs().max(), n
    norm = math.sqrt(sum(float(b.square().sum()) for b in want))
    got = list(got)
    assert abs(float(runtime.clip_grad_norm(got, 0.1 * norm)) - norm) <= 1e-4 * norm
    for n, a, b in zip(p, got, want):
        assert (a.double().cpu() - 0.1 * b).abs().max() <= 2e-4 * 0.1 * b.abs().max(), n


def test_a_captured_training_step(gpu):
    """Forward, backward, clipping and the update in one graph; each replay against eager."""
    def leaves(seed):
        return {n: t.cuda().requires_grad_() for n, t in weights(seed).items()}

    def step(p, tokens, s0):
        out, s = model(p, tokens[:, :-1], s0, *OWN)
        loss = loss_of(out, tokens[:, 1:]) + s.square().mean()
        grads = [g.contiguous() for g in torch.autograd.grad(loss, list(p.values()))]
        norm = runtime.clip_grad_norm(grads, 0.05)
        with torch.no_grad():
            for t, g in zip(p.values(), grads):
                t -= 0.5 * g
        return loss.detach(), norm

    held, (tokens, s0) = leaves(3), (t.cuda() for t in batch(4))
    tokens, s0 = tokens, s0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step({n: t.detach().clone().requires_grad_() for n, t in held.items()}, tokens, s0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        told = step(held, tokens, s0)
    for seed in (5, 6, 7):
        t, s = batch(seed)
        tokens.copy_(t)
        s0.copy_(s)
        own = {n: x.detach().clone().requires_grad_() for n, x in held.items()}
        graph.replay()
        want = step(own, tokens, s0)
        torch.cuda.synchronize()
        for a, b in zip(told, want):
            assert abs(float(a) - float(b)) <= 1e-5 * abs(float(b))
        for n in held:                      # torch's own sums may go in another order
            assert (held[n] - own[n]).abs().max() <= 1e-5 * own[n].abs().max(), n


def test_served(gpu):
    """A prompt, then token by token from its state: as feeding the whole text at once."""
    p = {n: t.cuda() for n, t in weights(2).items()}
    text = torch.randint(0, VOCAB, (4, 60), generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        whole, end = model(p, text, None, *OWN)
        logits, state = model(p, text[:, :40], None, *OWN)

        def step(q, k, v, g, s):
            return runtime.linear_step(q[:, 0], k[:, 0], v[:, 0], g, s)[:, None], s

        every = [logits]
        for t in range(40, 60):
            lg, state = model(p, text[:, t:t + 1], state, runtime.embed, runtime.layer_norm, step)
            every.append(lg)
    assert (whole - torch.cat(every, 1)).abs().max() <= 1e-4 * whole.abs().max()
    assert (end - state).abs().max() <= 1e-4 * end.abs().max()


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_the_default_type_changes_nothing(gpu, default):
    p = {n: t.cuda().requires_grad_() for n, t in weights(4).items()}
    tokens, s0 = (t.cuda() for t in batch(8))

    def run():
        x = runtime.embed(p["embed"], tokens[:, :-1], 2.0)
        q, k = x.reshape(3, 150, 2, 24), x.reshape(3, 150, 2, 24) * 0.1
        out, send = runtime.linear_attention(q, k, x.reshape(3, 150, 2, 24), p["g"][:2].neg().exp().neg())
        grads = torch.autograd.grad(out.square().sum() + send.sum(), [p["embed"], p["g"]])
        return out, send, *grads, runtime.grad_norm([g.contiguous() for g in grads])

    want = run()
    try:
        torch.set_default_dtype(default)
        have = run()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(have, want))


def test_embedding_beyond_32_bits(gpu):
    """Tables, batches and gradients of more than 2^31 elements, and the most rows of a sort."""
    gen = torch.Generator(gpu).manual_seed(5)
    R, D_, n = (1 << 21) + 333, 1032, (1 << 21) + 1001
    table = torch.empty(R, D_, dtype=torch.bfloat16, device=gpu).normal_(generator=gen)
    ids = torch.randint(0, R, (n,), device=gpu, generator=gen)
    ids[-1000:-500] = R - 1
    y = runtime.embed(table, ids)
    assert torch.equal(y[-1000:], table[ids[-1000:]]) and torch.equal(y[:1000], table[ids[:1000]])
    del y
    dy = torch.empty(n, D_, dtype=torch.bfloat16, device=gpu).normal_(generator=gen)
    grad = runtime.embed_bwd(dy, ids, R)
    for r in (R - 1, int(ids[7]), int(ids[-1])):
        at = (ids == r).nonzero()[:, 0]
        want, size = dy[at].double().sum(0), dy[at].double().abs().sum(0)
        room = 2.0 ** -8 * want.abs() + len(at) * 2.0 ** -24 * size + 2.0 ** -130
        assert bool(((grad[r].double() - want).abs() <= room).all()), r
    named = torch.zeros(R, dtype=torch.bool, device=gpu)
    named[ids] = True
    assert not grad[~named].any() and bool(grad[named].any(1).all())


def test_clipping_beyond_32_bits(gpu):
    gen = torch.Generator(gpu).manual_seed(6)
    n = (1 << 31) + 70001
    big = torch.empty(n, dtype=torch.bfloat16, device=gpu).normal_(0, 1e-3, generator=gen)
    xs = [big, torch.full((5,), 2.0, device=gpu)]
    want = math.sqrt(sum(float(x.double().square().sum()) for x in big.split(1 << 28)) + 20.0)
    tail = big[-100000:].double()
    norm = runtime.clip_grad_norm(xs, 0.5 * want)
    assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want
    f = 0.5 * want / (want + 1e-6)
    assert bool(((big[-100000:].double() - f * tail).abs() <= (2.0 ** -8 + 2.0 ** -22) * (f * tail).abs() + 2.0 ** -130).all())
