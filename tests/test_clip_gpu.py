"""The common norm of gradients and their clipping (runtime.grad_norm, clip_grad_norm)
against 64 bits.

Tolerances, fixed before the first run: the norm is a sum in 64 bits rounded once to fp32,
2^-24 (and 2^-40 for the order of the sum); a clipped value is an fp32 product by a factor
rounded to fp32, then rounded to T: 2 2^-24 + finfo(T).eps / 2 of the value, or half the
smallest number of T.
"""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def tensors(sizes, seed=0, kinds=(F32,), scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=g)).to(kinds[i % len(kinds)]).cuda() for i, n in enumerate(sizes)]


def norm64(xs):
    return math.sqrt(sum(float(x.double().square().sum()) for x in xs))


def check(xs, max_norm, ys, norm):
    want = norm64(xs)
    assert norm.shape == () and norm.dtype == F32
    assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want
    f = min(1.0, max_norm / (want + 1e-6))
    for x, y in zip(xs, ys):
        w = x.double() * f
        fi = torch.finfo(x.dtype)
        room = (fi.eps / 2 * (x.dtype != F32) + 2 * 2.0 ** -24) * w.abs() + fi.smallest_normal * fi.eps / 2
        assert y.dtype == x.dtype and ((y.double() - w).abs() <= room).all()


SIZES = [[1], [8191, 8192, 8193, 7], [0, 3, 0, 100000, 1], [5] * 300, [1 << 20, 333, 65536 * 3 + 1], [2 ** 24 + 5]]


@pytest.mark.parametrize("kinds", [(F32,), (BF16,), (F16,), (BF16, F32, F16)], ids=["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_against_64_bits(gpu, sizes, kinds):
    xs = tensors(sizes, len(sizes), kinds)
    want = norm64(xs)
    assert torch.equal(runtime.grad_norm(xs), runtime.grad_norm(xs))
    for bound in (0.25 * want, 4 * want, 0.0):
        ys = [torch.full_like(x, 9.0) for x in xs]
        norm = runtime.clip_grad_norm(xs, bound, out=ys)
        check(xs, bound, ys, norm)
        zs = [x.clone() for x in xs]
        again = runtime.clip_grad_norm(zs, bound)
        assert torch.equal(again, norm) and torch.equal(norm, runtime.grad_norm(xs))
        assert all(torch.equal(a, b) for a, b in zip(ys, zs))
    zs = [x.clone() for x in xs]
    runtime.clip_grad_norm(zs, 4 * want)
    assert all(torch.equal(a, b) for a, b in zip(xs, zs))


def test_unaligned_and_shaped(gpu):
    flat = torch.randn(100003).cuda().to(BF16)
    xs = [flat[1:5000].view(4999, 1), flat[5001:60000].view(3, -1)[:, 1:], flat[60002:]]
    xs[1] = xs[1].contiguous()
    out = torch.zeros_like(flat)
    ys = [out[:4999].view(4999, 1), out[5001:5001 + xs[1].numel()].view(xs[1].shape), out[60002:]]
    check(xs, 10.0, ys, runtime.clip_grad_norm(xs, 10.0, out=ys))
    zs = [x.clone() for x in xs]
    check(xs, 10.0, zs, runtime.clip_grad_norm(iter(zs), 10.0))


def test_sizes_of_values(gpu):
    """Squares that fp32 does not hold, and the smallest numbers."""
    for size in (1e30, 1e-30, 1e-42):
        xs = tensors([1000, 17], 3, scale=size)
        ys = [torch.empty_like(x) for x in xs]
        norm = runtime.clip_grad_norm(xs, size, out=ys)
        assert abs(float(norm) - norm64(xs)) <= 2.0 ** -24 * norm64(xs) + 2.0 ** -150
        if size > 1e-40:
            check(xs, size, ys, norm)


def test_not_finite(gpu):
    for bad in (math.inf, -math.inf, math.nan):
        xs = tensors([300, 5000], 4)
        xs[1][77] = bad
        ys = [torch.empty_like(x) for x in xs]
        norm = runtime.clip_grad_norm(xs, 1.0, out=ys)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and all(y.isnan().all() for y in ys)
        else:
            assert float(norm) == math.inf and not ys[0].any() and ys[1].isnan().sum() == 1


def test_versions_and_graphs(gpu):
    w = torch.randn(50, device="cuda", requires_grad=True)
    kept = torch.randn(50, device="cuda")
    y = (w * kept).sum()
    runtime.clip_grad_norm([kept], 1.0)
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()
    with pytest.raises(RuntimeError, match="leaf"):
        runtime.clip_grad_norm([w], 1.0)


def test_captured(gpu):
    """Replays follow the gradients' values, whatever ran between."""
    xs = tensors([70000, 33, 4096], 5, (BF16, F32))
    ys = [torch.empty_like(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        runtime.clip_grad_norm(xs, 3.0, out=ys)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = runtime.clip_grad_norm(xs, 3.0, out=ys)
    for i in range(4):
        for x, z in zip(xs, tensors([70000, 33, 4096], 10 + i, (BF16, F32), scale=0.001 * 30 ** i)):
            x.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        check(xs, 3.0, ys, norm)
        zs = [torch.empty_like(x) for x in xs]
        assert torch.equal(runtime.clip_grad_norm(xs, 3.0, out=zs), norm)
        assert all(torch.equal(a, b) for a, b in zip(ys, zs))


def test_one_tensor_twice(gpu):
    """Counts twice in a norm; as two gradients to scale, or as two places, it is refused."""
    x, y = tensors([3000], 6)[0], tensors([3000], 7)[0]
    assert abs(float(runtime.grad_norm([x, x, y])) - norm64([x, x, y])) <= (2.0 ** -24 + 2.0 ** -40) * norm64([x, x, y])
    kept = x.clone()
    for grads, out in (([x, x], None), ([x, x[10:20]], None), ([x, y], [y, x]), ([x], [x.view(-1)[0:0].new_empty(0)]),
                       ([x[:2000]], [x[1000:]]), ([y, y], [x, x])):
        with pytest.raises(ValueError):
            runtime.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(x, kept)
    a, b = torch.empty_like(x), torch.empty_like(x)
    check([x, x], 1.0, [a, b], runtime.clip_grad_norm([x, x], 1.0, out=[a, b]))


def test_two_streams_at_once(gpu):
    xs = [tensors([300000, 17, 9000], s, (BF16, F32)) for s in (8, 9)]
    want = []
    for x in xs:
        ys = [torch.empty_like(t) for t in x]
        want.append((runtime.clip_grad_norm(x, 2.0, out=ys), ys))
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                ys = [t.clone() for t in x]
                got.append((i, runtime.clip_grad_norm(ys, 2.0), ys))
    torch.cuda.synchronize()
    for i, norm, ys in got:
        assert torch.equal(norm, want[i][0]) and all(torch.equal(a, b) for a, b in zip(ys, want[i][1]))
