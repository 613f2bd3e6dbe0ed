"""The gated delta rule (runtime.gated_delta, delta_step) against its token-by-token
definition in 64 bits, forward and gradients.

Tolerances, fixed before the first run: an output of type T is one rounding
(finfo(T).eps / 2 of the value) away from a sum of fp32 precision. That sum runs over at
most K + 32 + 32 terms per product and four products deep per chunk, each addition off by
2^-24 of the sum of the terms' sizes, which is taken as the tensor's largest value:
4 (K + 64) 2^-24 for the forward, and four times that for gradients, whose products take
the forward's results. Products that only reach a 16-bit output hold their operands to
16 bits: 2^-16 of the terms' sizes more, with up to K + 32 terms of random sign: 2^-16 sqrt(K + 32).
"""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("q", "k", "v", "g", "beta", "s0")


def inputs(B, T, Hk, H, K, V, dtype, seed=0, N=None, dev="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    def unit(*s):
        x = rn(*s)
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-3)

    x = {"q": unit(B, T, Hk, K).to(dtype), "k": unit(B, T, Hk, K).to(dtype), "v": rn(B, T, H, V).to(dtype),
         "g": -torch.exp(rn(B, T, H) - 2), "beta": torch.sigmoid(2 * rn(B, T, H)),
         "s0": 0.3 * rn(B if N is None else N, H, K, V)}
    return {n: t.to(dev) for n, t in x.items()}


def ref(q, k, v, g, beta, s0, scale=None):
    """Token by token in 64 bits, on the CPU: (B,T,..) -> out, send (inputs are double)."""
    B, T, Hk, K = q.shape
    H = v.shape[2]
    rep, out, S = H // Hk, [], s0
    scale = K ** -0.5 if scale is None else scale
    for t in range(T):
        qt, kt = (x[:, t].repeat_interleave(rep, 1) for x in (q, k))
        S = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (S * kt[..., None]).sum(2))
        S = S + kt[..., None] * u[:, :, None, :]
        out.append(scale * (S * qt[..., None]).sum(2))
    return (torch.stack(out, 1) if out else v[:, :0]), S


def as64(x, grad=False):
    return [x[n].detach().double().cpu().requires_grad_(grad) for n in NAMES]


def close(name, x, y, K, grad=False):
    x, y = x.detach().double().cpu(), y.detach()
    assert x.shape == y.shape, name
    if not y.numel():
        return
    dt = close.dtype if name not in ("send", "dg", "dbeta", "ds0") else F32
    size = y.abs().max()
    tol = (16 if grad else 4) * (K + 64) * 2.0 ** -24 * size
    if name == "out" and dt != F32:
        tol = tol + 2.0 ** -16 * math.sqrt(K + 32) * size
    tol = tol + torch.finfo(dt).eps / 2 * y.abs()
    if dt == F16:
        tol = tol + 2.0 ** -25          # half a step of fp16's smallest values
    worst = ((x - y).abs() - tol).max()
    assert worst <= 0, f"{name}: {(x - y).abs().max():.3g} off, {size:.3g} large"


SHAPES = [  # B, T, Hk, H, K, V
    (1, 1, 1, 1, 1, 1), (2, 2, 1, 2, 3, 5), (1, 16, 2, 2, 64, 64), (1, 17, 1, 3, 64, 48), (2, 31, 2, 2, 40, 72),
    (1, 32, 1, 1, 128, 128), (3, 33, 1, 2, 65, 17), (1, 64, 2, 4, 128, 130), (2, 100, 1, 1, 127, 200),
    (1, 333, 3, 3, 24, 16), (1, 65, 1, 1, 8, 300),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(gpu, shape, dtype):
    close.dtype = dtype
    x = inputs(*shape, dtype)
    ro, rs = ref(*as64(x))
    out, send = runtime.gated_delta(**x)
    assert out.dtype == dtype and send.dtype == F32
    close("out", out, ro, shape[4])
    close("send", send, rs, shape[4])
    x["s0"] = None                      # no state: zeros
    out, send = runtime.gated_delta(**x, scale=0.7)
    x["s0"] = torch.zeros_like(rs).float()
    ro, rs = ref(*as64(x), scale=0.7)
    close("out", out, ro, shape[4])
    close("send", send, rs, shape[4])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(gpu, shape, dtype):
    close.dtype = dtype
    x = inputs(*shape, dtype, seed=1)
    gen = torch.Generator().manual_seed(2)
    x64 = as64(x, True)
    ro, rs = ref(*x64)
    do = torch.randn(ro.shape, generator=gen).to(dtype)
    ds = torch.randn(rs.shape, generator=gen)
    want = torch.autograd.grad((ro, rs), x64, (do.double(), ds.double()))
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf)
    got = torch.autograd.grad((out, send), leaf, (do.cuda(), ds.cuda()), retain_graph=True)
    close("out", out, ro, shape[4])
    for n, a, b in zip(NAMES, got, want):
        assert a.dtype == x[n].dtype
        close("d" + n, a, b, shape[4], True)
    again = torch.autograd.grad((out, send), leaf, (do.cuda(), ds.cuda()), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "the same call gave other bits"
    # only one of the two outputs is used
    for keep, outs in ((0, (do, None)), (1, (None, ds))):
        got1 = torch.autograd.grad((out, send)[keep], leaf, outs[keep].cuda(), retain_graph=True)
        z = torch.zeros_like
        both = torch.autograd.grad((out, send), leaf, (do.cuda() if keep == 0 else z(out),
                                                       ds.cuda() if keep == 1 else z(send)), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got1, both))


def test_gradients_against_differences(gpu):
    """<gradient, direction> of the fp32 kernels against central differences of the
    64-bit definition: the difference's own error is of order h^2 = 1e-10."""
    x = inputs(2, 70, 1, 2, 24, 20, F32, seed=3)
    gen = torch.Generator().manual_seed(4)
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf)
    do, ds = (torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (out, send))
    do, ds = do.float(), ds.float()
    got = torch.autograd.grad((out, send), leaf, (do.cuda(), ds.cuda()))
    base = as64(x)

    def loss(v):
        o, s = ref(*v)
        return float((o * do.double()).sum() + (s * ds.double()).sum())

    for i, n in enumerate(NAMES):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        plus, minus = ([b + s * h * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
        want = (loss(plus) - loss(minus)) / (2 * h)
        have = float((got[i].double().cpu() * d).sum())
        size = float(got[i].double().norm().cpu() * d.norm())
        assert abs(want - have) <= 1e-5 * size, n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_packed_sequences_equal_their_own_calls(gpu, dtype):
    lens = [1, 32, 33, 0, 5, 64, 100, 0, 17, 2]
    pad_front, pad_back = 3, 7
    T = sum(lens) + pad_front + pad_back
    x = inputs(1, T, 2, 4, 48, 40, dtype, N=len(lens))
    edges = [pad_front]
    for n in lens:
        edges.append(edges[-1] + n)
    cu = torch.tensor(edges, dtype=torch.int32, device="cuda")
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf, cu_seqlens=cu)
    do, ds = torch.randn_like(out), torch.randn_like(send)
    got = torch.autograd.grad((out, send), leaf, (do, ds))
    assert not out[:, :pad_front].any() and not out[:, T - pad_back:].any()
    for g in got[:5]:
        assert not g[:, :pad_front].any() and not g[:, T - pad_back:].any()
    for i, n in enumerate(lens):
        a, e = edges[i], edges[i + 1]
        if n == 0:
            assert torch.equal(send[i], x["s0"][i]) and torch.equal(got[5][i], ds[i])
            continue
        one = [x[m].detach()[:, a:e].clone().requires_grad_() for m in NAMES[:5]]
        one.append(x["s0"].detach()[i:i + 1].clone().requires_grad_())
        o, s = runtime.gated_delta(*one)
        assert torch.equal(o[0], out[0, a:e]) and torch.equal(s[0], send[i])
        gr = torch.autograd.grad((o, s), one, (do[:, a:e], ds[i:i + 1]))
        for m, p, q in zip(NAMES, gr, got):
            assert torch.equal(p[0], q[i] if m == "s0" else q[0, a:e]), m


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 4100, 1, 1, 8, 5), (1, 5003, 1, 2, 65, 40), (2, 4200, 1, 1, 128, 20)], ids=str)
def test_long_sequences_in_parts(gpu, shape, dtype):
    """Few heads and thousands of tokens: the sequence is scanned in parts that are joined.
    A part's map is one more product of K terms than the scan's own, once a part."""
    close.dtype = dtype
    x = inputs(*shape, dtype, seed=21)
    x["g"] *= 0.01                         # states that reach through several parts
    x64 = as64(x, True)
    ro, rs = ref(*x64)
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf)
    close("out", out, ro, shape[4])
    close("send", send, rs, shape[4])
    with torch.no_grad():
        plain = runtime.gated_delta(*leaf)
    assert torch.equal(plain[0], out) and torch.equal(plain[1], send)
    gen = torch.Generator().manual_seed(22)
    do, ds = torch.randn(ro.shape, generator=gen).to(dtype), torch.randn(rs.shape, generator=gen)
    want = torch.autograd.grad((ro, rs), x64, (do.double(), ds.double()))
    got = torch.autograd.grad((out, send), leaf, (do.cuda(), ds.cuda()))
    for n, a, b in zip(NAMES, got, want):
        close("d" + n, a, b, shape[4], True)


def test_long_packed_sequences_in_parts(gpu):
    close.dtype = F32
    lens = [3000, 1, 4000, 0, 700, 2500]
    x = inputs(1, sum(lens), 1, 2, 24, 16, F32, N=len(lens), seed=23)
    x["g"] *= 0.01
    edges = torch.tensor([0] + lens).cumsum(0)
    out, send = runtime.gated_delta(**x, cu_seqlens=edges.int().cuda())
    for i, n in enumerate(lens):
        a, e = int(edges[i]), int(edges[i + 1])
        one = {m: (x[m][:, a:e] if m != "s0" else x[m][i:i + 1]) for m in NAMES}
        ro, rs = ref(*as64(one))
        if n:
            close("out", out[:, a:e], ro, 24)
        close("send", send[i:i + 1], rs, 24)


def test_edges_outside_the_rows_are_clamped(gpu):
    x = inputs(1, 50, 1, 1, 16, 16, F32, N=2)
    for edges, same in (([-5, 20, 1000], [0, 20, 50]), ([0, 50, 50], [0, 50, 50])):
        a, b = (runtime.gated_delta(**x, cu_seqlens=torch.tensor(e, dtype=torch.int32, device="cuda"))
                for e in (edges, same))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
def test_strided_views_equal_copies(gpu, dtype):
    """q, k and v as slices of one projection, at odd offsets and with other axis orders."""
    B, T, H, K, V = 2, 45, 3, 24, 20
    x = inputs(B, T, H, H, K, V, dtype)
    wide = torch.randn(B, T, H, 2 * K + V + 1, device="cuda").to(dtype)
    wide[..., 1:1 + K], wide[..., 1 + K:1 + 2 * K], wide[..., 1 + 2 * K:] = x["q"], x["k"], x["v"]
    views = dict(x, q=wide[..., 1:1 + K], k=wide[..., 1 + K:1 + 2 * K], v=wide[..., 1 + 2 * K:])
    heads = dict(x, **{n: x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in "qkv"})
    last = dict(x, **{n: x[n].transpose(2, 3).contiguous().transpose(2, 3) for n in "qkv"})
    want = runtime.gated_delta(**x)
    for y in (views, heads, last):
        got = runtime.gated_delta(**y)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    first = {n: t[:, 0] for n, t in x.items() if n != "s0"}
    s1, s2 = x["s0"].clone(), x["s0"].clone()
    o1 = runtime.delta_step(*(t.contiguous() for t in first.values()), s1)
    o2 = runtime.delta_step(*(views[n][:, 0] for n in ("q", "k", "v", "g", "beta")), s2)
    assert torch.equal(o1, o2) and torch.equal(s1, s2)


@pytest.mark.parametrize("case", ["forget", "strong", "far", "no_write", "full_write", "same_keys"])
@pytest.mark.parametrize("T", [9, 75])
def test_hard_values(gpu, case, T):
    close.dtype = F32
    x = inputs(1, T, 1, 2, 32, 24, F32, seed=5)
    if case == "forget":               # exp(g) = 0: the state begins anew
        x["g"][:, 3], x["g"][:, 5, 0], x["g"][:, T - 1, 1] = -math.inf, -math.inf, -math.inf
    elif case == "strong":
        x["g"] *= 300
    elif case == "far":                # nearly no decay after one that leaves nothing
        x["g"].fill_(-1e-4)
        x["g"][:, 2] = -1e30
    elif case == "no_write":
        x["beta"].zero_()
    elif case == "full_write":
        x["beta"].fill_(1.0)
    else:                              # every write meets all the earlier ones
        x["k"] = x["k"][:, :1].expand(-1, T, -1, -1).contiguous()
        x["beta"].fill_(1.0)
        x["g"].fill_(0.0)
    leaf = [x[n].requires_grad_() for n in NAMES]
    x64 = as64(x, True)
    ro, rs = ref(*x64)
    out, send = runtime.gated_delta(*leaf)
    close("out", out, ro, 32)
    close("send", send, rs, 32)
    do, ds = torch.randn(ro.shape), torch.randn(rs.shape)
    want = torch.autograd.grad((ro, rs), x64, (do.double(), ds.double()))
    got = torch.autograd.grad((out, send), leaf, (do.cuda(), ds.cuda()))
    for n, a, b in zip(NAMES, got, want):
        if n == "g":                   # at -inf the definition's own gradient is 0 times infinity or 0
            b = torch.where(torch.isfinite(b), b, 0.0)
        close("d" + n, a, b, 32, True)


def test_nan_stays_in_its_sequence_and_head(gpu):
    x = inputs(2, 80, 2, 2, 16, 16, F32)
    want = runtime.gated_delta(**x)
    x["v"][0, 40, 1] = math.nan
    x["g"][0, 70, 1] = math.inf
    out, send = runtime.gated_delta(**x)
    assert out[0, 40:, 1].isnan().all() and send[0, 1].isnan().all()
    assert torch.equal(out[0, :32], want[0][0, :32])           # the chunks before it
    assert torch.equal(out[0, :, 0], want[0][0, :, 0]) and torch.equal(out[1], want[0][1])
    assert torch.equal(send[0, 0], want[1][0, 0]) and torch.equal(send[1], want[1][1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 2, 4, 64, 64), (2, 1, 3, 128, 128), (1, 12, 12, 64, 64),
                                   (5, 2, 2, 100, 37), (2, 1, 1, 65, 300)], ids=str)
def test_step(gpu, shape, dtype):
    close.dtype = dtype
    B, Hk, H, K, V = shape
    x = inputs(B, 3, Hk, H, K, V, dtype, seed=6)
    ro, rs = ref(*as64(x))
    s = x["s0"].clone()
    for t in range(3):
        args = [x[n][:, t] for n in NAMES[:5]]
        new = torch.full_like(s, math.nan)
        apart = runtime.delta_step(*args, s, send=new)
        out = runtime.delta_step(*args, s)
        assert torch.equal(out, apart) and torch.equal(s, new)
        close("out", out, ro[:, t], K)
    close("send", s, rs, K)


def test_prompt_then_steps_equal_one_prompt(gpu):
    close.dtype = F32
    x = inputs(2, 90, 2, 2, 64, 64, F32, seed=7)
    ro, rs = ref(*as64(x))
    out, s = runtime.gated_delta(*(x[n][:, :80] for n in NAMES[:5]), x["s0"])
    outs = [out] + [runtime.delta_step(*(x[n][:, t] for n in NAMES[:5]), s)[:, None] for t in range(80, 90)]
    close("out", torch.cat(outs, 1), ro, 64)
    close("send", s, rs, 64)


def test_views_that_the_kernels_do_not_take_are_copied(gpu):
    """Expanded axes (stride 0) are read in place; a token stride of 2^24 is copied."""
    x = inputs(2, 40, 1, 2, 16, 16, F32, seed=30)
    same = dict(x, q=x["q"][:, :1].expand(-1, 40, -1, -1), k=x["k"][:1].expand(2, -1, -1, -1))
    want = runtime.gated_delta(**{n: t.clone() for n, t in same.items()})
    got = runtime.gated_delta(**same)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    far = torch.zeros(2, 3, 1 << 24, dtype=F16, device="cuda")
    half = {n: t[:, :3].half() if n in "qkv" else t[:, :3].contiguous() if n != "s0" else t for n, t in x.items()}
    far[:, :, :16] = half["q"][:, :, 0]
    view = far[:, :, None, :16]
    assert view.stride(1) == 1 << 24
    a, b = runtime.gated_delta(**half), runtime.gated_delta(**dict(half, q=view))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_second_derivatives_are_refused(gpu):
    x = inputs(1, 20, 1, 1, 8, 8, F32)
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, _ = runtime.gated_delta(*leaf)
    grad, = torch.autograd.grad(out.sum(), leaf[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_two_streams_at_once(gpu):
    """Calls on two streams share nothing: each has the results of a call alone."""
    xs = [inputs(2, 300, 1, 2, 64, 64, BF16, seed=40 + i) for i in range(2)]
    want = [runtime.gated_delta(**x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                got.append(runtime.gated_delta(**x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_tokens_and_no_sequences(gpu):
    x = inputs(2, 0, 1, 2, 8, 8, F32)
    out, send = runtime.gated_delta(**x)
    assert out.shape == (2, 0, 2, 8) and torch.equal(send, x["s0"])
    leaf = [x[n].requires_grad_() for n in NAMES]
    out, send = runtime.gated_delta(*leaf)
    ds = torch.randn_like(send)
    got = torch.autograd.grad(send, leaf, ds)
    assert torch.equal(got[5], ds) and got[0].shape == x["q"].shape
    x = inputs(0, 5, 1, 2, 8, 8, F32)
    out, send = runtime.gated_delta(**x)
    assert out.shape == (0, 5, 2, 8) and send.shape == (0, 2, 8, 8)
    assert runtime.delta_step(*(x[n][:, 0] for n in NAMES[:5]), x["s0"]).shape == (0, 2, 8)


def test_on_another_stream_and_in_a_graph(gpu):
    x = inputs(2, 70, 1, 2, 32, 32, BF16, seed=8)
    leaf = [x[n].requires_grad_() for n in NAMES]
    do = torch.randn(2, 70, 2, 32, device="cuda").to(BF16)
    want = runtime.gated_delta(*leaf)
    wgrad = torch.autograd.grad(want[0], leaf, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = runtime.gated_delta(*leaf)
        grad = torch.autograd.grad(got[0], leaf, do)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip((*want, *wgrad), (*got, *grad)))
    plain = [x[n].detach().clone() for n in NAMES]
    state = plain[5]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, send = runtime.delta_fwd(*plain)[:2]
        token = runtime.delta_step(*(t[:, 0] for t in plain[:5]), send)
    for seed in (9, 10, 11):
        y = inputs(2, 70, 1, 2, 32, 32, BF16, seed=seed)
        for p, n in zip(plain, NAMES):
            p.copy_(y[n])
        graph.replay()
        o, s = runtime.gated_delta(*plain)
        tok = runtime.delta_step(*(t[:, 0] for t in plain[:5]), s)
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(s, send) and torch.equal(tok, token)
    assert state is plain[5]


def test_backward_in_a_graph(gpu):
    """Forward and backward captured together, replayed on other inputs."""
    x = inputs(1, 64, 1, 2, 32, 32, F32, seed=12)
    plain = [x[n] for n in NAMES]
    do, ds = torch.randn(1, 64, 2, 32, device="cuda"), torch.randn_like(x["s0"])

    def both():
        out, send, saved = runtime.delta_fwd(*plain, keep=True)
        return out, send, *runtime.delta_bwd(*plain, saved, do, ds)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (13, 14, 15):
        y = inputs(1, 64, 1, 2, 32, 32, F32, seed=seed)
        for p, n in zip(plain, NAMES):
            p.copy_(y[n])
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
