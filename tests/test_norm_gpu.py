"""Layer norm (runtime.layer_norm) against its formula in 64 bits, forward and gradients.

Tolerances, fixed before the first run. With h the normalised row, values are of size
|h w| + |b|; the mean and the variance are sums of D values in a tree (16 values in a lane,
then at most 10 levels), so each carries at most 32 roundings of 2^-24 of the sum of sizes
and h at most 40 2^-24 (|h| + |mean| rstd + |h|^2 ...): 64 2^-24 of (1 + |mean| rstd + |h|).
The result is rounded once to its type (eps / 2). dx is a difference of three such terms of
size rstd (|dy w| + rms(dy w) (1 + |h|)). Column sums over R rows hold at most R / 1024 + 64 + 24
additions in a chain.
"""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def rows(R, D, dtype, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, D, generator=g) * (0.1 + torch.rand(R, 1, generator=g)) + mean * torch.randn(R, 1, generator=g))
    w, b = 1 + 0.2 * torch.randn(D, generator=g), 0.2 * torch.randn(D, generator=g)
    dy = torch.randn(R, D, generator=g)
    return x.to(dtype).cuda(), w.cuda(), b.cuda(), dy.to(dtype).cuda()


def formula(x, w, b, dy, eps):
    x, w, b, dy = (t.double().cpu() for t in (x, w, b, dy))
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + eps)
    h, e = (x - m) * r, dy * w
    dx = r * (e - e.mean(1, keepdim=True) - h * (e * h).mean(1, keepdim=True))
    return h, m, r, e, h * w + b, dx, (dy * h).sum(0), dy.sum(0)


def check(x, w, b, dy, eps, got, dtype):
    h, m, r, e, y, dx, dw, db = formula(x, w, b, dy, eps)
    R = x.shape[0]
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    unit = 64 * U * (1 + (m * r).abs() + h.abs())
    tol_y = unit * w.double().cpu().abs() + 4 * U * b.double().cpu().abs() + half * y.abs() + tiny
    rms = e.square().mean(1, keepdim=True).sqrt()
    tol_dx = 4 * unit * r * (e.abs() + 2 * rms * (1 + h.abs())) + half * dx.abs() + tiny
    chain = (R / 1024 + 64 + 24) * U
    d = dy.double().cpu().abs()
    tol_dw = chain * (d * h.abs()).sum(0) + (d * unit).sum(0)
    tol_db = chain * d.sum(0)
    for n, a, want, tol in zip(("y", "dx", "dw", "db"), got, (y, dx, dw, db), (tol_y, tol_dx, tol_dw, tol_db)):
        if a is not None:
            off = (a.detach().double().cpu() - want).abs()
            assert (off <= tol).all(), f"{n}: {off.max():.3g} off"


def run(x, w, b, dy, eps):
    leaf = [t.requires_grad_() for t in (x, w, b)]
    y = runtime.layer_norm(*leaf, eps)
    return y, *torch.autograd.grad(y, leaf, dy)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [1, 2, 7, 8, 63, 200, 511, 512, 520, 1000, 1024, 1030, 1536, 2048, 2055, 4096, 5000,
                               8192, 9999, 16384])
def test_norm(gpu, D, dtype):
    dt = DT[dtype]
    for R in (1, 5, 67):
        x, w, b, dy = rows(R, D, dt, seed=D + R)
        eps = 4.1e-4
        got = run(x, w, b, dy, eps)
        assert got[0].dtype == got[1].dtype == dt and got[2].dtype == torch.float32
        check(x, w, b, dy, eps, got, dt)


def test_many_rows(gpu):
    x, w, b, dy = rows(9001, 24, torch.float32)
    got = run(x, w, b, dy, 1e-5)
    check(x, w, b, dy, 1e-5, got, torch.float32)
    again = run(x, w, b, dy, 1e-5)
    assert all(torch.equal(a, c) for a, c in zip(got, again)), "the same call gave other bits"


def test_a_mean_far_from_zero(gpu):
    """The variance comes from the centred values: |mean| rstd is about 1000 here."""
    x, w, b, dy = rows(9, 777, torch.float32, mean=300.0)
    check(x, w, b, dy, 1e-5, run(x, w, b, dy, 1e-5), torch.float32)


def test_constant_rows_and_without_weights(gpu):
    x = torch.full((4, 96), 2.5, device="cuda")
    assert not runtime.layer_norm(x).any()
    x, w, b, dy = rows(6, 130, torch.bfloat16)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    x.requires_grad_()
    y = runtime.layer_norm(x)
    want = runtime.layer_norm(x, one, zero)
    assert torch.equal(y, want)
    assert torch.equal(*(torch.autograd.grad(t, x, dy)[0] for t in (y, want)))
    w.requires_grad_()
    y = runtime.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    check(x, w, zero, dy, 1e-5, (y, gx, gw, None), torch.bfloat16)


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True)])
def test_only_the_gradients_asked_for(gpu, need):
    x, w, b, dy = rows(33, 300, torch.float32)
    y, mean, rstd = runtime.norm_fwd(x, w, b, 1e-5, keep=True)
    whole = runtime.norm_bwd(dy, x, w, mean, rstd)
    for n, a, c in zip(need, runtime.norm_bwd(dy, x, w, mean, rstd, need=need), whole):
        assert torch.equal(a, c) if n else a is None


def test_against_differences(gpu):
    """Directional derivative against central differences of the formula in 64 bits."""
    x, w, b, dy = rows(12, 50, torch.float32, seed=3)
    got = run(x, w, b, dy, 1e-3)[1:]
    base = [t.detach().double().cpu() for t in (x, w, b)]
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        v = [float((formula(*[t + (s * 1e-5 * d if j == i else 0) for j, t in enumerate(base)], dy, 1e-3)[4]
                    * dy.double().cpu()).sum()) for s in (1, -1)]
        have = float((got[i].double().cpu() * d).sum())
        assert abs((v[0] - v[1]) / 2e-5 - have) <= 1e-5 * float(got[i].double().norm().cpu() * d.norm())


def test_views_offsets_and_nan(gpu):
    x, w, b, dy = rows(20, 64, torch.bfloat16)
    want = runtime.layer_norm(x, w, b)
    wide = torch.zeros(20, 100, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:67] = x
    assert torch.equal(runtime.layer_norm(wide[:, 3:67], w, b), want)
    flat = torch.zeros(20 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = x.reshape(-1)                      # rows at odd addresses
    assert torch.equal(runtime.layer_norm(flat[1:].view(4, 5, 64), w, b).view(20, 64), want)
    x[7, 5] = float("nan")
    got = runtime.layer_norm(x, w, b)
    assert got[7].isnan().all()
    keep = torch.arange(20, device="cuda") != 7
    assert torch.equal(got[keep], want[keep])
    assert runtime.layer_norm(x[:0], w, b).shape == (0, 64)
    e = x[:0].detach().requires_grad_()
    g = torch.autograd.grad(runtime.layer_norm(e, w.requires_grad_()), (e, w), dy[:0])
    assert g[0].shape == (0, 64) and not g[1].any()


def test_in_a_graph(gpu):
    x, w, b, dy = rows(300, 264, torch.float16)
    run(x, w, b, dy, 1e-5)
    x, w, b = (t.detach() for t in (x, w, b))

    def both():
        y, mean, rstd = runtime.norm_fwd(x, w, b, 1e-5, keep=True)
        return y, *runtime.norm_bwd(dy, x, w, mean, rstd)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in range(3):
        for t, v in zip((x, w, b, dy), rows(300, 264, torch.float16, seed=seed)):
            t.copy_(v)
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, want))
