"""The three operators together, as a pre-normed recurrent language model of one block
uses them: trained (layer norm, gated delta rule, their gradients through plain torch
layers) against the same model in 64 bits, and served (prompt, then token by token in a
captured graph: norm, delta step, head, sampled token) against its own prompt form.

Tolerances, fixed before the first run. The model's matrices are fp32 torch products of
at most 64 terms, the operators hold fp32; a gradient passes about ten such stages, each
off by at most some 64 2^-24 = 4e-6 of the sizes involved: 1e-4 of the largest entry.
"""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
D, Hk, H, K, V, VOCAB = 48, 2, 4, 16, 24, 97


def weights(seed=0):
    g = torch.Generator().manual_seed(seed)

    def rn(*s, std=0.2):
        return std * torch.randn(*s, generator=g)

    return {"embed": rn(VOCAB, D, std=1.0), "w1": 1 + rn(D), "b1": rn(D), "qk": rn(2 * Hk * K, D), "v": rn(H * V, D),
            "gb": rn(2 * H, D), "out": rn(D, H * V), "w2": 1 + rn(D), "b2": rn(D)}


def delta64(q, k, v, g, beta, s):
    outs = []
    for t in range(q.shape[1]):
        qt, kt = (x[:, t].repeat_interleave(H // Hk, 1) for x in (q, k))
        s = s * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (s * kt[..., None]).sum(2))
        s = s + kt[..., None] * u[:, :, None, :]
        outs.append((s * qt[..., None]).sum(2) * K ** -0.5)
    return torch.stack(outs, 1), s


def norm64(x, w, b, eps):
    d = x - x.mean(-1, keepdim=True)
    return d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * w + b


def model(p, tokens, s0, norm, delta):
    """tokens (B, T) -> logits (B, T, VOCAB), state."""
    B, T = tokens.shape
    x = p["embed"][tokens]
    h = norm(x, p["w1"], p["b1"], 4.1e-4)
    q, k = (h @ p["qk"].t()).view(B, T, 2, Hk, K).unbind(2)
    k = k / k.norm(dim=-1, keepdim=True)
    v = (h @ p["v"].t()).view(B, T, H, V)
    g, beta = (h @ p["gb"].t()).view(B, T, 2, H).unbind(2)
    o, s = delta(q, k, v, -torch.nn.functional.softplus(g), torch.sigmoid(beta), s0)
    x = x + o.reshape(B, T, H * V) @ p["out"].t()
    return norm(x, p["w2"], p["b2"], 4.1e-4) @ p["embed"].t(), s


def loss_of(logits, targets):
    z = logits - logits.logsumexp(-1, keepdim=True)
    return -z.gather(-1, targets[..., None]).mean()


def test_trained(gpu):
    p = weights()
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, VOCAB, (3, 78), generator=g)
    s0 = 0.1 * torch.randn(3, H, K, V, generator=g)
    p64 = {n: t.double().requires_grad_() for n, t in p.items()}
    lg, s = model(p64, tokens[:, :-1], s0.double(), norm64, delta64)
    want = torch.autograd.grad(loss_of(lg, tokens[:, 1:]) + s.square().mean(), list(p64.values()))
    pd = {n: t.cuda().requires_grad_() for n, t in p.items()}
    td = tokens.cuda()
    out, sd = model(pd, td[:, :-1], s0.cuda(), runtime.layer_norm, runtime.gated_delta)
    got = torch.autograd.grad(loss_of(out, td[:, 1:]) + sd.square().mean(), list(pd.values()))
    assert (out.double().cpu() - lg).abs().max() <= 1e-4 * lg.abs().max()
    assert (sd.double().cpu() - s).abs().max() <= 1e-4 * s.abs().max()
    for n, a, b in zip(p, got, want):
        assert (a.double().cpu() - b).abs().max() <= 1e-4 * b.abs().max(), n


def test_served(gpu):
    """A prompt, then sampled tokens one by one in a captured graph. Feeding the whole
    text as one prompt gives the same logits, and with them the same tokens wherever the
    random number is not at a border of the distribution."""
    p = {n: t.cuda() for n, t in weights(2).items()}
    B, T, N = 4, 37, 20
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, VOCAB, (B, T), generator=g).cuda()
    u = torch.rand(N, B, dtype=torch.float64, generator=g).cuda()
    pick = dict(temperature=0.9, top_k=30, top_p=0.9, min_p=0.001)

    def step(q, k, v, gg, beta, s):
        return runtime.delta_step(q[:, 0], k[:, 0], v[:, 0], gg[:, 0].contiguous(), beta[:, 0].contiguous(), s)[:, None], s

    logits, state = model(p, prompt, None, runtime.layer_norm, runtime.gated_delta)
    token = runtime.sample_tokens(logits[:, -1], u[0], **pick)
    text, every = [token.clone()], [logits[:, -1].clone()]
    now = torch.empty_like(u[0])
    # warm the library calls up on the side stream that the graph is captured from
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model(p, token[:, None].long(), state.clone(), runtime.layer_norm, step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, _ = model(p, token[:, None].long(), state, runtime.layer_norm, step)
        token.copy_(runtime.sample_tokens(held[:, 0], now, **pick))
    for i in range(1, N):
        now.copy_(u[i])
        graph.replay()
        torch.cuda.synchronize()
        text.append(token.clone())
        every.append(held[:, 0].clone())
    text, every = torch.stack(text, 1), torch.stack(every, 1)
    whole, end = model(p, torch.cat([prompt, text[:, :-1].long()], 1), None, runtime.layer_norm, runtime.gated_delta)
    assert (whole[:, T - 1:] - every).abs().max() <= 1e-4 * whole.abs().max()
    assert (end - state).abs().max() <= 1e-4 * end.abs().max()
    for i in range(N):
        assert torch.equal(runtime.sample_tokens(every[:, i], u[i], **pick), text[:, i])


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_the_default_type_changes_nothing(gpu, default):
    """Workspaces, statistics and gradients of decays are fp32 whatever torch's default is."""
    gen = torch.Generator().manual_seed(3)

    def rn(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float32).cuda()

    q, k, v = rn(2, 77, 2, 16), rn(2, 77, 2, 16) / 4, rn(2, 77, 4, 24)
    leaves = [q, k, v, -rn(2, 77, 4).abs(), torch.sigmoid(rn(2, 77, 4)), rn(2, 4, 16, 24), rn(24), rn(24)]
    seed = rn(2, 77, 4, 24)

    def run():
        own = [t.clone().requires_grad_() for t in leaves]
        out, send = runtime.gated_delta(*own[:6])
        y = runtime.layer_norm(out, *own[6:])
        return y, send, *torch.autograd.grad([y, send], own, [seed, leaves[5]])

    want = run()
    try:
        torch.set_default_dtype(default)
        have = run()
    finally:
        torch.set_default_dtype(torch.float32)
    for a, b in zip(have, want):
        assert a.dtype == torch.float32 and torch.equal(a, b)


def test_what_the_forward_kept_for_other_shapes_is_refused(gpu):
    x = [torch.zeros(1, 40, 2, 16, device="cuda") for _ in range(3)]
    g, beta = torch.zeros(2, 1, 40, 2, device="cuda")
    short = runtime.delta_fwd(*(t[:, :20] for t in x), g[:, :20], beta[:, :20], keep=True)[2]
    for saved in (short, None, (None, None)):
        with pytest.raises(ValueError, match="saved"):
            runtime.delta_bwd(*x, g, beta, None, saved, x[2])


def test_training_in_a_graph(gpu):
    """Forward and autograd's backward captured after a pass on a side stream whose outputs
    are still alive; replays against eager passes over copies of the leaves."""
    gen = torch.Generator().manual_seed(5)

    def leaves():
        r = [torch.randn(*s, generator=gen).cuda() for s in
             [(2, 70, 2, 16), (2, 70, 2, 16), (2, 70, 4, 24), (2, 70, 4), (2, 70, 4), (2, 4, 16, 24), (24,), (24,)]]
        return [r[0], r[1] / 4, r[2], -r[3].abs(), torch.sigmoid(r[4]), *r[5:]]

    def run(t):
        out, send = runtime.gated_delta(*t[:6])
        y = runtime.layer_norm(out, *t[6:])
        torch.autograd.backward([y, send], [dy, ds])
        return y, send

    dy, ds = torch.randn(2, 70, 4, 24, generator=gen).cuda(), torch.randn(2, 4, 16, 24, generator=gen).cuda()
    held = [t.requires_grad_() for t in leaves()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = run(held)
    torch.cuda.current_stream().wait_stream(side)
    for t in held:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run(held)
    for _ in range(3):
        new = [t.requires_grad_() for t in leaves()]
        with torch.no_grad():
            for t, n in zip(held, new):
                t.copy_(n)
        graph.replay()
        want = run(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(held, new))
    del warm


def test_a_capture_beside_a_living_eager_graph_is_refused(gpu):
    x = torch.randn(3, 24, device="cuda", requires_grad=True)
    q, k, v = (torch.randn(1, 40, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    g, beta = -torch.rand(1, 40, 2, device="cuda"), torch.rand(1, 40, 2, device="cuda")
    calls = [lambda: runtime.layer_norm(x), lambda: runtime.gated_delta(q, k, v, g, beta)[0]]
    for call in calls:
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="still alive"):
                call()
            torch.zeros(1, device="cuda")
        want = torch.autograd.grad(alive.sum(), x if call is calls[0] else q)[0]
        assert torch.isfinite(want).all()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
