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


def ref(q, k, v, g, beta, s0, scale):
    """Token by token in 64 bits, on the CPU."""
    q, k, v, g, beta, S = (x.double().cpu() for x in (q, k, v, g, beta, s0))
    rep, outs = v.shape[2] // q.shape[2], []
    for t in range(q.shape[1]):
        qt, kt = (x[:, t].repeat_interleave(rep, 1) for x in (q, k))
        S = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (S * kt[..., None]).sum(2))
        S = S + kt[..., None] * u[:, :, None, :]
        outs.append(scale * (S * qt[..., None]).sum(2))
    return torch.stack(outs, 1), S


@pytest.mark.parametrize("case", ["state", "writes", "products"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_sums_hold_fp32_before_a_16_bit_output(gpu, dtype, case):
    """1 + 2^-9 + 2^-20 less 1 + 2^-9, as an entry of the state, a write, or a product of query
    and key: an operand cut to 16 bits would lose the 2^-20 that is left. The sums are of size
    1 and have at most eight terms: 8 2^-24, half of what is left."""
    T, K, V, wide = 20, 8, 16, 1 + 2.0 ** -9 + 2.0 ** -20
    x = {"q": torch.zeros(1, T, 1, K), "k": torch.zeros(1, T, 1, K), "v": torch.zeros(1, T, 1, V),
         "g": torch.zeros(1, T, 1), "beta": torch.zeros(1, T, 1), "s0": torch.zeros(1, 1, K, V)}
    x["q"][..., :6] = 1
    if case == "state":
        x["s0"][0, 0, 0], x["s0"][0, 0, 1] = wide, -(1 + 2.0 ** -9)
    elif case == "writes":
        x["k"][0, 0, 0, 0] = x["k"][0, 1, 0, 1] = 1
        x["v"][0, 0], x["v"][0, 1] = 1, -1
        x["beta"][0, 0], x["beta"][0, 1] = wide, 1 + 2.0 ** -9
    else:
        x["k"][0, 0, 0, :3] = torch.tensor([1, 2.0 ** -9, 2.0 ** -20])
        x["k"][0, 1, 0, 3:5] = torch.tensor([1, 2.0 ** -9])
        x["v"][0, 0], x["v"][0, 1] = 1, -1
        x["beta"][0, :2] = 1
    x = {n: t.cuda().to(dtype if n in "qkv" else torch.float32) for n, t in x.items()}
    want = ref(*(x[n] for n in NAMES), 1.0)[0]
    assert (want[0, 2:] == 2.0 ** -20).all()
    got = runtime.gated_delta(**x, scale=1.0)[0].double().cpu()
    off = float((got - want)[0, 2:].abs().max())
    assert off <= 8 * 2.0 ** -24


LENS = [1, 32, 33, 0, 5, 64, 100, 0, 17, 2]


def test_packed_fp16_sequences_equal_their_own_calls(gpu):
    edges = torch.tensor([0] + LENS).cumsum(0) + 3
    T = int(edges[-1]) + 7
    for K, V in ((48, 40), (128, 72)):
        x = inputs(1, T, 2, 4, K, V, torch.float16, 61, N=len(LENS))
        leaf = [x[n].requires_grad_() for n in NAMES]
        out, send = runtime.gated_delta(*leaf, cu_seqlens=edges.int().cuda())
        gen = torch.Generator().manual_seed(62)
        do, ds = (torch.randn(t.shape, generator=gen).to(t.dtype).cuda() for t in (out, send))
        got = torch.autograd.grad((out, send), leaf, (do, ds))
        for t in (out, *got[:5]):
            assert not t[:, :3].any() and not t[:, T - 7:].any()
        for i, n in enumerate(LENS):
            a, e = int(edges[i]), int(edges[i + 1])
            if n == 0:
                assert torch.equal(send[i], x["s0"][i]) and torch.equal(got[5][i], ds[i])
                continue
            one = [t.detach()[:, a:e].clone().requires_grad_() for t in leaf[:5]]
            one.append(leaf[5].detach()[i:i + 1].clone().requires_grad_())
            o, s = runtime.gated_delta(*one)
            assert torch.equal(o[0], out[0, a:e]) and torch.equal(s[0], send[i])
            for m, p, q in zip(NAMES, torch.autograd.grad((o, s), one, (do[:, a:e], ds[i:i + 1])), got):
                assert torch.equal(p[0], q[i] if m == "s0" else q[0, a:e]), m
