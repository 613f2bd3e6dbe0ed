"""Linear attention where it can go wrong: parts of long sequences, graphs and streams,
values that are not finite, the ends of its sizes, arrays of more than 2^31 elements.
Tolerances as in test_linear_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime
from test_linear_gpu import BF16, F16, F32, NAMES, close, forward_close, gradients_close, inputs, ref

pytestmark = pytest.mark.gpu


def run(leaf, dout, dsend, **kw):
    leaf = [t.detach().requires_grad_() for t in leaf]
    out, send = runtime.linear_attention(*leaf, **kw)
    return out.detach(), send.detach(), *torch.autograd.grad((out, send), leaf, (dout, dsend))


@pytest.mark.parametrize("head_g", [False, True], ids=["token_g", "head_g"])
def test_gradients_against_differences(gpu, head_g):
    """Along a direction d of one input: the result is linear in each of q, k, v and s0, so a
    central difference is exact but for rounding; in g its error is step^2 / 6 of a third
    derivative, of the size of the first (decays of up to 3 tokens' reach): 1e-2 for steps of
    0.1. Each loss is off by at most 4 (D + 64) 2^-24 of the sum of its terms' sizes, which the
    difference divides by the step."""
    B, T, Hk, H, K, V = 2, 100, 1, 2, 24, 40
    x = inputs(B, T, Hk, H, K, V, F32, seed=5, head_g=head_g)
    gen = torch.Generator().manual_seed(6)
    wo, ws = (torch.randn(*s, generator=gen).cuda() for s in ((B, T, H, V), (B, H, K, V)))

    def loss(y):
        out, send = runtime.linear_attention(*(y[n] for n in NAMES))
        o, s = out.double() * wo, send.double() * ws
        return float(o.sum() + s.sum()), float(o.abs().sum() + s.abs().sum())

    grads = dict(zip(NAMES, run([x[n] for n in NAMES], wo, ws)[2:]))
    for n in NAMES:
        step = 0.1 if n == "g" else 1.0
        d = torch.randn(x[n].shape, generator=gen).cuda() * (0.1 if n == "g" else 1.0)
        (a, size), (b, _) = loss({**x, n: x[n] + step * d}), loss({**x, n: x[n] - step * d})
        want = float((grads[n].double() * d).sum())
        room = 4 * (K + V + 64) * 2.0 ** -24 * size / step + (1e-2 * float((grads[n] * d).abs().sum()) if n == "g" else 0)
        assert abs((a - b) / (2 * step) - want) <= room, n


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 1000, 1, 1, 64, 64), (1, 641, 2, 2, 128, 200), (3, 514, 1, 3, 20, 36),
                                   (40, 70, 2, 4, 32, 32), (1, 3000, 2, 4, 33, 17)], ids=str)
def test_parts(gpu, shape, dtype):
    """Sequences that are cut into parts, of whole and of broken chunks."""
    B, T, Hk, H, K, V = shape
    x = inputs(*shape, dtype, seed=T)
    gen = torch.Generator().manual_seed(1)
    dout, dsend = torch.randn(B, T, H, V, generator=gen).to(dtype).cuda(), torch.randn(B, H, K, V, generator=gen).cuda()
    out, send, *got = run([x[n] for n in NAMES], dout, dsend)
    forward_close(x, out, send)
    gradients_close(x, got, dout, dsend)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_the_same_call_gives_the_same_bits(gpu, dtype):
    x = inputs(2, 700, 1, 4, 40, 56, dtype, seed=2, head_g=True)
    dout, dsend = torch.randn(2, 700, 4, 56).cuda().to(dtype), torch.randn(2, 4, 40, 56).cuda()
    a, b = (run([x[n] for n in NAMES], dout, dsend) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_views_equal_copies(gpu):
    """Any strides, a misaligned first element, a gradient that is a view."""
    B, T, H, K, V = 2, 130, 2, 32, 48
    for dtype in (F32, BF16, F16):
        gen = torch.Generator().manual_seed(3)
        wide = torch.randn(B, T, 3 + H * (2 * K + V), generator=gen).to(dtype).cuda()[..., 3:]
        q, k, v = wide.split([H * K, H * K, H * V], -1)
        g = -torch.rand(H, B, T, generator=gen).cuda().permute(1, 2, 0)
        views = [q.view(B, T, H, K), k.view(B, T, H, K), v.view(B, T, H, V), g, torch.randn(B, H, V, K).cuda().transpose(2, 3)]
        dout = torch.randn(B, V, H, T, generator=gen).to(dtype).cuda().permute(0, 3, 2, 1)
        dsend = torch.randn(B, H, V, K).cuda().transpose(2, 3)
        a = run(views, dout, dsend)
        b = run([t.contiguous() for t in views], dout.contiguous(), dsend.contiguous())
        assert all(torch.equal(p, r) for p, r in zip(a, b))


def test_broadcast_inputs(gpu):
    """Heads, tokens and batches that share one row; their gradients are the sums."""
    B, T, H, K, V = 2, 75, 3, 16, 24
    gen = torch.Generator().manual_seed(4)
    base = [torch.randn(1, 1, 1, K, generator=gen), 0.2 * torch.randn(1, T, 1, K, generator=gen),
            torch.randn(B, 1, H, V, generator=gen), -torch.rand(B, 1, 1, generator=gen), torch.randn(1, 1, K, V, generator=gen)]
    base = [t.cuda().requires_grad_() for t in base]
    sizes = [(B, T, H, K), (B, T, H, K), (B, T, H, V), (B, T, H), (B, H, K, V)]
    wide = [t.expand(s) for t, s in zip(base, sizes)]
    out, send = runtime.linear_attention(*wide)
    got = torch.autograd.grad(out.square().sum() + send.sum(), base)
    d = [t.detach().double().cpu().requires_grad_() for t in base]
    o, s = ref(*(t.expand(n) for t, n in zip(d, sizes)))
    close(out.detach(), o.detach(), F32, 4 * 88 * 2.0 ** -24, "out")
    want = torch.autograd.grad(o.square().sum() + s.sum(), d)
    for n, a, b in zip(NAMES, got, want):          # sums of up to B T H V such gradients
        close(a, b, F32, 8 * 88 * 2.0 ** -24 * math.sqrt(T * H), "d" + n)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["q", "k", "v", "g", "s0"])
def test_what_is_not_finite_stays_in_its_sequence_and_head(gpu, where, bad):
    if where == "g" and bad == -math.inf:
        pytest.skip("forgets the state: a number")
    B, T, H, K, V, at = 2, 200, 3, 24, 24, 130
    x = inputs(B, T, H, H, K, V, F32, seed=6)
    want = runtime.linear_attention(*(x[n] for n in NAMES))
    if where == "s0":
        x["s0"][1, 2, 3, 4] = bad
    else:
        x[where][1, at, 2] = bad
    out, send = runtime.linear_attention(*(x[n] for n in NAMES))
    keep = torch.ones(B, T, H, dtype=torch.bool)
    keep[1, (0 if where == "s0" else at // 64 * 64):, 2] = False
    assert torch.equal(out[keep.cuda()], want[0][keep.cuda()])
    assert not torch.isfinite(out[1, at, 2]).all()
    same = torch.ones(B, H, dtype=torch.bool)
    same[1, 2] = False
    assert torch.equal(send[same.cuda()], want[1][same.cuda()])
    if where != "q":
        assert not torch.isfinite(send[1, 2]).all()


@pytest.mark.parametrize("case", ["state", "products"])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
def test_sums_hold_fp32_before_a_16_bit_output(gpu, dtype, case):
    """1 + 2^-9 + 2^-20 less 1 + 2^-9, as entries of the state or products of query and key: an
    operand cut to 16 bits would lose the 2^-20 that is left. The sums are of size 1 and have
    at most eight terms: 8 2^-24, half of what is left."""
    T, K, V, wide = 20, 8, 16, 1 + 2.0 ** -9 + 2.0 ** -20
    x = {"q": torch.zeros(1, T, 1, K), "k": torch.zeros(1, T, 1, K), "v": torch.zeros(1, T, 1, V),
         "g": torch.zeros(1, T, 1), "s0": torch.zeros(1, 1, K, V)}
    x["q"][..., :6] = 1
    if case == "state":
        x["s0"][0, 0, 0], x["s0"][0, 0, 1] = wide, -(1 + 2.0 ** -9)
    else:
        x["k"][0, 0, 0, :3] = torch.tensor([1, 2.0 ** -9, 2.0 ** -20])
        x["k"][0, 1, 0, 3:5] = torch.tensor([1, 2.0 ** -9])
        x["v"][0, 0], x["v"][0, 1] = 1, -1
    x = {n: t.cuda().to(dtype if n in "qkv" else F32) for n, t in x.items()}
    want = ref(*(x[n].double().cpu() for n in NAMES), 1.0)[0]
    assert (want[0, 2:] == 2.0 ** -20).all()
    got = runtime.linear_attention(**x, scale=1.0)[0].double().cpu()
    assert float((got - want)[0, 2:].abs().max()) <= 8 * 2.0 ** -24


def test_growth(gpu):
    """g above 0 is not what is meant, but a number."""
    x = inputs(1, 150, 1, 2, 16, 16, F32, seed=7)
    x["g"] = 0.05 * torch.randn(1, 150, 2, generator=torch.Generator().manual_seed(1)).cuda()
    out, send = runtime.linear_attention(*(x[n] for n in NAMES))
    forward_close(x, out, send)


def test_edges_outside_the_rows_are_clamped(gpu):
    x = inputs(1, 90, 1, 2, 16, 16, F32, seed=8, N=2)
    wild = torch.tensor([-50, 40, 1000], dtype=torch.int32, device="cuda")
    tame = torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
    a, b = (runtime.linear_attention(*(x[n] for n in NAMES), cu_seqlens=cu) for cu in (wild, tame))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_no_tokens_and_no_sequences(gpu):
    for B, T in ((2, 0), (0, 5), (0, 0)):
        x = inputs(B, T, 1, 2, 8, 8, F32)
        out, send, *grads = run([x[n] for n in NAMES], torch.zeros(B, T, 2, 8).cuda(), torch.ones(B, 2, 8, 8).cuda())
        assert out.shape == (B, T, 2, 8) and torch.equal(send, x["s0"])
        assert all(torch.equal(a, torch.zeros_like(a)) for a in grads[:4]) and torch.equal(grads[4], torch.ones_like(send))


def test_second_derivatives_and_a_tracked_state_are_refused(gpu):
    x = inputs(1, 20, 1, 1, 8, 8, F32)
    q = x["q"].requires_grad_()
    out, _ = runtime.linear_attention(q, x["k"], x["v"], x["g"])
    (dq,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)
    one = [x[n].detach()[:, 0] for n in "qkvg"]
    s = torch.zeros(1, 1, 8, 8, device="cuda")
    w = torch.ones_like(s).requires_grad_()
    read = (s * w).sum()
    runtime.linear_step(*one, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        read.backward()
    flat = torch.zeros(200, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        runtime.linear_step(*one, flat[:64].view(1, 1, 8, 8), send=flat[4:68].view(1, 1, 8, 8))


def test_what_the_forward_kept_for_other_shapes_is_refused(gpu):
    x = inputs(1, 600, 1, 1, 16, 16, F32)
    args = [x[n] for n in NAMES]
    out, send, parts = runtime.linear_fwd(*args, keep=True)
    assert parts is not None
    for bad in (None, parts[:-4], parts.double()):
        with pytest.raises(ValueError, match="parts"):
            runtime.linear_bwd(*args, send, bad, out)
    with pytest.raises(ValueError, match="send"):
        runtime.linear_bwd(*args, send[0], parts, out)


def test_two_streams_at_once(gpu):
    xs = [inputs(2, 500, 1, 2, 64, 64, BF16, seed=s) for s in (1, 2)]
    dout, dsend = torch.randn(2, 500, 2, 64).cuda().to(BF16), torch.randn(2, 2, 64, 64).cuda()
    want = [run([x[n] for n in NAMES], dout, dsend) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(run([x[n] for n in NAMES], dout, dsend))
    torch.cuda.synchronize()
    for w, all_ in zip(want, got):
        for one in all_:
            assert all(torch.equal(a, b) for a, b in zip(w, one))


def test_two_graphs(gpu):
    """Two captured training passes and a captured step share nothing: replayed in turn, each
    with new inputs, against eager calls."""
    xs = [inputs(2, 300, 1, 2, 32, 32, BF16, seed=s) for s in (1, 2)]
    dout, dsend = torch.randn(2, 300, 2, 32).cuda().to(BF16), torch.randn(2, 2, 32, 32).cuda()
    side = torch.cuda.Stream()
    graphs = []
    for x in xs:
        plain = [x[n] for n in NAMES]

        def both(plain=plain):
            out, send, parts = runtime.linear_fwd(*plain, keep=True)
            grads = runtime.linear_bwd(*plain, send, parts, dout, dsend)
            return out, send, *grads, runtime.linear_step(*(t[:, 0] for t in plain[:4]), send.clone())

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        graphs.append((graph, plain, both, held))
    for seed in (3, 4, 5):
        for i, (graph, plain, both, held) in enumerate(graphs):
            y = inputs(2, 300, 1, 2, 32, 32, BF16, seed=10 * seed + i)
            for p, n in zip(plain, NAMES):
                p.copy_(y[n])
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, plain, both, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, both()))


def test_a_capture_beside_a_living_eager_graph_is_refused(gpu):
    q, k, v = (torch.randn(1, 40, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    g = -torch.rand(2, device="cuda")
    table = torch.randn(9, 16, device="cuda", requires_grad=True)
    ids = torch.arange(9, device="cuda")
    for call in (lambda: runtime.linear_attention(q, k, v, g)[0], lambda: runtime.embed(table, ids)):
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="still alive"):
                call()
            torch.zeros(1, device="cuda")
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 40, 1, 2, 128, 4096), (1, 34, 5, 65535, 1, 1), (65535, 14, 1, 1, 2, 3),
                                   (65535, 2, 1, 1, 4, 4)], ids=str)
def test_at_its_largest(gpu, shape, dtype):
    B, T, Hk, H, K, V = shape
    x = {n: t.cpu() for n, t in inputs(*shape, dtype, seed=1).items()}
    x64 = [x[n].double().to(gpu).requires_grad_() for n in NAMES]
    ro, rs = ref(*x64)
    gen = torch.Generator().manual_seed(2)
    do, ds = torch.randn(ro.shape, generator=gen).to(dtype).to(gpu), torch.randn(rs.shape, generator=gen).to(gpu)
    want = torch.autograd.grad((ro, rs), x64, (do.double(), ds.double()))
    out, send, *got = run([x[n].to(gpu) for n in NAMES], do, ds)
    with torch.no_grad():
        plain = runtime.linear_attention(*(x[n].to(gpu) for n in NAMES))
    D = max(K, V)
    for n, a, b, grad in (("out", out, ro, 1), ("send", send, rs, 1), ("plain", plain[0], ro, 1), ("end", plain[1], rs, 1),
                          *(("d" + n, a, b, 2 if n != "g" else 2 * math.sqrt(T)) for n, a, b in zip(NAMES, got, want))):
        tol = 4 * grad * (D + 64) * 2.0 ** -24 * b.abs().max() + torch.finfo(a.dtype).eps / 2 * b.abs()
        assert float(((a.detach().double() - b.detach()).abs() - tol.detach()).max()) <= 0, n


def test_beyond_32_bits(gpu):
    """More than 2^31 values in v, out and their gradients. The state is forgotten at a token
    near the end: from there on the results are those of the last tokens' own call, to
    rounding (the parts lie differently)."""
    T, H, K, V = 136000, 128, 64, 128
    at = T - 500
    assert T * H * V > 1 << 31
    gen = torch.Generator(gpu).manual_seed(3)
    bf = dict(dtype=BF16, device=gpu)
    q, k = (torch.empty(1, T, 1, K, **bf).normal_(0, K ** -0.5, generator=gen) for _ in range(2))
    v, dout = (torch.empty(1, T, H, V, **bf).normal_(generator=gen) for _ in range(2))
    g = -0.2 * torch.rand(1, T, H, device=gpu, generator=gen)
    g[:, at] = -math.inf
    ones = torch.ones(1, H, K, V, device=gpu)
    s0 = torch.zeros_like(ones)
    whole = run([q, k, v, g, s0], dout, ones)
    tail = run([t[:, at:].clone() for t in (q, k, v, g)] + [s0], dout[:, at:].clone(), ones)
    tol = 8 * (128 + 64) * 2.0 ** -24
    for n, a, b in zip(("out", "send", "q", "k", "v", "g"), whole, tail):
        a = (a[:, at:] if n != "send" else a).double()
        b = b.double()
        half = torch.finfo(whole[0].dtype).eps if n in ("out", "q", "k", "v") else 0
        slack = 2 * math.sqrt(500) if n == "g" else 1
        # q's and k's gradients are sums over 128 heads
        size = b.abs().max() * (math.sqrt(H) if n in "qk" else 1) * slack
        if n == "g":
            a, b = a[:, 1:], b[:, 1:]              # the forgetting one's is 0 but for what cancels
        assert float(((a - b).abs() - tol * size - half * b.abs()).max()) <= 0, n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_packed_with_a_decay_per_head(gpu, dtype):
    """Parts of packed sequences, shared heads, V in more than one block; dg sums over all."""
    edges, T, Hk, H, K, V = [0, 1, 300, 300, 1030], 1030, 1, 2, 20, 136
    spans = list(zip(edges, edges[1:]))
    x = inputs(1, T, Hk, H, K, V, dtype, seed=8, N=len(spans), head_g=True)
    leaf = [x[n].clone().requires_grad_() for n in NAMES]
    out, send = runtime.linear_attention(*leaf, cu_seqlens=torch.tensor(edges, dtype=torch.int32, device="cuda"))
    forward_close(x, out, send, parts=spans)
    dout, dsend = torch.randn_like(out), torch.randn_like(send)
    got = torch.autograd.grad((out, send), leaf, (dout, dsend))

    def packed(q, k, v, g, s0):
        res = [ref(q[:, a:e], k[:, a:e], v[:, a:e], g, s0[i:i + 1]) for i, (a, e) in enumerate(spans)]
        return torch.cat([r[0] for r in res], 1), torch.cat([r[1] for r in res])

    gradients_close(x, got, dout, dsend, packed)


def test_states_off_16_bytes(gpu):
    """States that begin four bytes past an aligned address equal aligned ones, bit for bit."""
    for B, T, H, K, V in ((3, 1, 2, 64, 32), (2, 700, 2, 32, 64), (1, 40, 3, 128, 100)):
        x = inputs(B, T, H, H, K, V, F32, seed=T)
        off = torch.empty(x["s0"].numel() + 1, device="cuda")[1:].view(x["s0"].shape).copy_(x["s0"])
        dout, dsend = torch.randn(B, T, H, V).cuda(), torch.randn(B, H, K, V).cuda()
        doff = torch.empty(dsend.numel() + 1, device="cuda")[1:].view(dsend.shape).copy_(dsend)
        plain = [x[n] for n in NAMES[:4]]
        assert all(torch.equal(a, b) for a, b in zip(run([*plain, x["s0"]], dout, dsend), run([*plain, off], dout, doff)))
        one = [t[:, 0] for t in plain]
        a, b = x["s0"].clone(), off
        assert torch.equal(runtime.linear_step(*one, a), runtime.linear_step(*one, b)) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("head_g", [False, True], ids=["token_g", "head_g"])
@pytest.mark.parametrize("edges", [[3, 10, 90], [0, 1], [7, 7], [0, 0, 700], [150, 150, 151, 699]], ids=str)
def test_tokens_of_no_sequence_are_cleared(gpu, monkeypatch, edges, head_g, dtype):
    """Whatever the outputs' memory held before; rows of odd sizes. Against the call without
    those tokens, whose sums differ by twice their tolerance, and each is rounded once more:
    finfo(T).eps / 2 of its value beside close's own."""
    T, Hk, H, K, V = 700, 1, 3, 5, 7
    x = inputs(1, T, Hk, H, K, V, dtype, seed=T, N=len(edges) - 1, head_g=head_g)
    cu = torch.tensor(edges, dtype=torch.int32, device="cuda")
    dout, dsend = torch.randn(1, T, H, V).cuda().to(dtype), torch.randn(len(edges) - 1, H, K, V).cuda()
    live = torch.zeros(T, dtype=torch.bool, device="cuda")
    live[edges[0]:edges[-1]] = True
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(77))
    out, send, *grads = run([x[n] for n in NAMES], dout, dsend, cu_seqlens=cu)
    for t in (out, *grads[:3], *([] if head_g else grads[3:4])):
        assert not t[0, ~live].any()
    part = {n: t if n == "s0" or t.dim() == 1 else t[:, live] for n, t in x.items()}
    if live.any():
        near = run([part[n] for n in NAMES], dout[:, live], dsend, cu_seqlens=cu - edges[0])
        for a, b in zip((out, *grads[:3]), (near[0], *near[2:5])):
            close(a[:, live], b.double().cpu(), dtype,
                  16 * (7 + 64) * 2.0 ** -24 + torch.finfo(dtype).eps / 2 * (dtype != F32), "a shifted call")
