"""Linear attention with a decay for each head (runtime.linear_attention, linear_step)
against its definition in 64 bits, forward and gradients.

Tolerances, fixed before the first run. An output of type T is one rounding
(finfo(T).eps / 2 of the value) away from a sum of fp32 precision. Such a sum runs over at
most D = max(K, V) terms through the state and 64 of its chunk, whose own terms are sums of
D: each addition is off by 2^-24 of the terms' sizes, taken as the tensor's largest value
(times 4, since terms cancel): 4 (D + 64) 2^-24. Gradients take such results as operands:
twice that. The decay's gradient adds up to L tokens' differences q.dq - k.dk, of errors
of random sign, from the largest of the two: 4 (D + 64) 2^-24 sqrt(L) of that.
"""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("q", "k", "v", "g", "s0")


def inputs(B, T, Hk, H, K, V, dtype, seed=0, N=None, head_g=False):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    g = -torch.exp(rn(H) - 2) if head_g else -torch.exp(rn(B, T, H) - 2)
    x = {"q": rn(B, T, Hk, K).to(dtype), "k": (rn(B, T, Hk, K) * K ** -0.5).to(dtype), "v": rn(B, T, H, V).to(dtype),
         "g": g, "s0": 0.3 * rn(B if N is None else N, H, K, V)}
    return {n: t.cuda() for n, t in x.items()}


def ref(q, k, v, g, s0, scale=None):
    """Token by token in 64 bits, on the CPU (inputs are double)."""
    B, T, Hk, K = q.shape
    H = v.shape[2]
    g, out, S = g.expand(B, T, H), [], s0
    scale = K ** -0.5 if scale is None else scale
    for t in range(T):
        qt, kt = (x[:, t].repeat_interleave(H // Hk, 1) for x in (q, k))
        S = S * torch.exp(g[:, t])[..., None, None] + kt[..., None] * v[:, t, :, None, :]
        out.append(scale * (S * qt[..., None]).sum(2))
    return torch.stack(out, 1) if out else v * 0, S


def close(got, want, dtype, tol, what):
    got, want = got.double().cpu(), want.double()
    size = float(want.abs().max()) if want.numel() else 0.0
    room = torch.finfo(dtype).eps / 2 * want.abs() * (dtype != F32) + tol * size + 1e-30
    assert got.shape == want.shape, what
    worst = ((got - want).abs() / room).max() if want.numel() else 0.0
    assert worst <= 1, f"{what}: {float(worst):.2f} of the tolerance"


def forward_close(x, out, send, scale=None, parts=None):
    d = {n: t.detach().double().cpu() for n, t in x.items()}
    K, V = x["q"].shape[-1], x["v"].shape[-1]
    tol = 4 * (max(K, V) + 64) * 2.0 ** -24
    if parts is None:
        o, s = ref(*(d[n] for n in NAMES), scale=scale)
    else:
        res = []
        for i, (a, e) in enumerate(parts):
            g = d["g"] if d["g"].dim() == 1 else d["g"][:, a:e]
            res.append(ref(d["q"][:, a:e], d["k"][:, a:e], d["v"][:, a:e], g, d["s0"][i:i + 1], scale=scale))
        o = torch.zeros(*d["v"].shape, dtype=torch.float64)
        for (a, e), (oo, _) in zip(parts, res):
            o[:, a:e] = oo
        s = torch.cat([r[1] for r in res])
    close(out.detach(), o, x["v"].dtype, tol, "out")
    close(send.detach(), s, F32, tol, "send")


SHAPES = [  # B, T, Hk, H, K, V
    (1, 1, 1, 1, 1, 1), (2, 13, 2, 4, 16, 24), (1, 64, 1, 1, 64, 64), (1, 65, 2, 2, 64, 64), (2, 130, 1, 3, 40, 72),
    (1, 300, 2, 2, 128, 128), (1, 257, 1, 2, 128, 64), (2, 100, 3, 3, 64, 128), (1, 97, 1, 1, 33, 300), (3, 31, 2, 2, 7, 5),
    (1, 1100, 1, 1, 128, 130),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("head_g", [False, True], ids=["token_g", "head_g"])
def test_forward_and_gradients(gpu, shape, dtype, head_g):
    x = inputs(*shape, dtype, seed=sum(shape), head_g=head_g)
    B, T, Hk, H, K, V = shape
    with torch.no_grad():
        out, send = runtime.linear_attention(*(x[n] for n in NAMES))
    forward_close(x, out, send)
    gen = torch.Generator().manual_seed(9)
    dout = torch.randn(B, T, H, V, generator=gen).to(dtype).cuda()
    dsend = torch.randn(B, H, K, V, generator=gen).cuda()
    leaf = [x[n].clone().requires_grad_() for n in NAMES]
    out, send = runtime.linear_attention(*leaf)
    forward_close(x, out, send)
    got = torch.autograd.grad((out, send), leaf, (dout, dsend))
    gradients_close(x, got, dout, dsend)


def gradients_close(x, got, dout, dsend, ref_of=ref):
    d = {n: x[n].detach().double().cpu().requires_grad_() for n in NAMES}
    o, s = ref_of(*(d[n] for n in NAMES))
    want = dict(zip(NAMES, torch.autograd.grad((o, s), [d[n] for n in NAMES], (dout.double().cpu(), dsend.double().cpu()))))
    got = dict(zip(NAMES, got))
    D, T = max(x["q"].shape[-1], x["v"].shape[-1]), x["q"].shape[1]
    tol = 8 * (D + 64) * 2.0 ** -24
    for n in ("q", "k", "v", "s0"):
        close(got[n], want[n], x[n].dtype, tol, "d" + n)
    size = max(float((d[n] * want[n]).detach().sum(-1).abs().max()) for n in ("q", "k"))
    size = max(size, float((s * dsend.double().cpu()).detach().sum((-1, -2)).abs().max()))
    many = x["q"].shape[0] * T if x["g"].dim() == 1 else 1
    room = 4 * (D + 64) * 2.0 ** -24 * math.sqrt(T) * size * many
    worst = float((got["g"].double().cpu() - want["g"]).abs().max()) / room
    assert got["g"].dtype == F32 and worst <= 1, f"dg: {worst:.2f} of the tolerance"


def test_scale_no_state_and_one_gradient(gpu):
    x = inputs(2, 70, 1, 2, 24, 40, F32, seed=3)
    x["s0"] = torch.zeros_like(x["s0"])
    out, send = runtime.linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.37)
    forward_close(x, out, send, scale=0.37)
    v = x["v"].clone().requires_grad_()
    out, send = runtime.linear_attention(x["q"], x["k"], v, x["g"])
    (dv,) = torch.autograd.grad(send.square().sum(), v)      # no gradient of out
    d = {n: t.double().cpu() for n, t in x.items()}
    d["v"].requires_grad_()
    (want,) = torch.autograd.grad(ref(*(d[n] for n in NAMES))[1].square().sum(), d["v"])
    close(dv, want, F32, 8 * 104 * 2.0 ** -24, "dv")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("edges", [[0, 5, 5, 70, 900], [0, 0, 0, 1], [3, 67, 131, 700, 1000], [0, 64, 128, 1024]],
                         ids=str)
def test_packed(gpu, edges, dtype):
    """Sequences end to end, empty ones and tokens of none among them."""
    T, H, Hk, K, V = 1024, 4, 2, 48, 64
    n = len(edges) - 1
    x = inputs(1, T, Hk, H, K, V, dtype, seed=n, N=n)
    cu = torch.tensor(edges, dtype=torch.int32, device="cuda")
    spans = list(zip(edges, edges[1:]))
    out, send = runtime.linear_attention(*(x[m] for m in NAMES), cu_seqlens=cu)
    forward_close(x, out, send, parts=spans)
    live = torch.zeros(T, dtype=torch.bool)
    for a, e in spans:
        live[a:e] = True
    assert not out[0, ~live.cuda()].any()
    leaf = [x[m].clone().requires_grad_() for m in NAMES]
    out, send = runtime.linear_attention(*leaf, cu_seqlens=cu)
    dout, dsend = torch.randn_like(out), torch.randn_like(send)
    got = torch.autograd.grad((out, send), leaf, (dout, dsend))

    def packed(q, k, v, g, s0):
        res = [ref(q[:, a:e], k[:, a:e], v[:, a:e], g[:, a:e], s0[i:i + 1]) for i, (a, e) in enumerate(spans)]
        o = torch.cat([v[:, :edges[0]] * 0] + [r[0] for r in res] + [v[:, edges[-1]:] * 0], 1)
        return o, torch.cat([r[1] for r in res])

    gradients_close(x, got, dout * live[None, :, None, None].cuda(), dsend, packed)
    for t in got[:4]:
        assert not t[0, ~live.cuda()].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 12, 12, 64, 64), (5, 2, 4, 128, 100), (3, 1, 3, 9, 33), (2, 1, 1, 1, 1)], ids=str)
@pytest.mark.parametrize("head_g", [False, True], ids=["token_g", "head_g"])
def test_step(gpu, shape, dtype, head_g):
    B, Hk, H, K, V = shape
    x = inputs(B, 1, Hk, H, K, V, dtype, seed=K, head_g=head_g)
    one = {n: t if n == "s0" or t.dim() == 1 else t[:, 0] for n, t in x.items()}
    send = torch.empty_like(x["s0"])
    out = runtime.linear_step(*(one[n] for n in NAMES), send=send)
    forward_close(x, out[:, None], send)
    s = x["s0"].clone()
    again = runtime.linear_step(one["q"], one["k"], one["v"], one["g"], s)
    assert torch.equal(again, out) and torch.equal(s, send)


def test_steps_continue_a_prompt(gpu):
    x = inputs(2, 45, 2, 2, 32, 48, F32, seed=4)
    out, send = runtime.linear_attention(*(x[n][:, :40] if n != "s0" else x[n] for n in NAMES))
    outs = [out]
    for t in range(40, 45):
        outs.append(runtime.linear_step(*(x[n][:, t] for n in "qkvg"), send)[:, None])
    forward_close(x, torch.cat(outs, 1), send)


@pytest.mark.parametrize("T", [11, 50, 300])
def test_forgetting(gpu, T):
    """-inf forgets all before, exactly; -200 and less are 0 in fp32 too."""
    x = inputs(1, T, 1, 2, 16, 16, F32, seed=T)
    x["g"][:, T // 2] = -math.inf
    x["g"][:, T // 2 + 1, 1] = -500.0
    y = {n: t.clone() for n, t in x.items()}
    for n in "qkv":
        y[n][:, :T // 2] += 1.0
    y["s0"] += 2.0
    a, b = (runtime.linear_attention(*(z[n] for n in NAMES)) for z in (x, y))
    assert torch.equal(a[0][:, T // 2:], b[0][:, T // 2:]) and torch.equal(a[1], b[1])
    z = {n: t if n == "s0" else t[:, T // 2:] for n, t in x.items()}
    z["g"] = z["g"].clamp_min(-200.0)
    forward_close(z, a[0][:, T // 2:], a[1])


def test_strides_and_alignment(gpu):
    """Views of one projection's output, an odd column first; rows of other strides."""
    B, T, H, K, V = 2, 75, 3, 24, 40
    for dtype in (F32, BF16):
        wide = torch.randn(B, T, 1 + H * (2 * K + V), device="cuda").to(dtype)
        q, k, v = wide[..., 1:].split([H * K, H * K, H * V], -1)
        x = {"q": q.view(B, T, H, K), "k": 0.2 * k.view(B, T, H, K), "v": v.view(B, T, H, V),
             "g": -torch.rand(B, H, T, device="cuda").transpose(1, 2), "s0": torch.randn(B, H, K, V, device="cuda")}
        out, send = runtime.linear_attention(*(x[n] for n in NAMES))
        forward_close(x, out, send)
        y = dict(x, k=x["k"][:, :1].expand(B, T, H, K), q=x["q"].transpose(1, 2).contiguous().transpose(1, 2))
        out, send = runtime.linear_attention(*(y[n] for n in NAMES))
        forward_close(y, out, send)
        leaf = [y[n].detach().requires_grad_() for n in NAMES]
        out, send = runtime.linear_attention(*leaf)
        dout = torch.randn(B, V, T, H, device="cuda").to(dtype).permute(0, 2, 3, 1)
        dsend = torch.randn_like(send)
        gradients_close(y, torch.autograd.grad((out, send), leaf, (dout, dsend)), dout, dsend)
