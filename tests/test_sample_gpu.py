"""Sampling on the device (runtime.sample_tokens) against its definition in 64 bits
(numpy, row by row) and against the scheduler's host sampler. Tokens have to be equal:
random numbers closer than 1e-9 to a border of the distribution are moved away from it
beforehand (the kernel's weights are whole multiples of 2^-42 of the largest or finer,
so a row's running shares are off by less than 2^20 2^-42 = 2.4e-7 only if every token
weighs as much as the largest; for the rows here by less than 1e-9)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from sunnynet_amd import runtime
from sunnynet_amd.runtime.serve import sample_logits

pytestmark = pytest.mark.gpu


def weights(row, t, k, p, m):
    """The kept weights of one row in index order (float64)."""
    z = row / t
    w = np.exp(z - z.max())
    if 0 < k < z.size:
        w[z < np.sort(z)[-k]] = 0.0
    if 0 < p < 1:
        order = np.argsort(-z, kind="stable")
        ws = w[order]
        before = np.cumsum(ws) - ws
        cut = before > p * ws.sum()
        cut[0] = False
        w[order[cut]] = 0.0
    w[w < m] = 0.0
    return w


def pick(row, u, t, k, p, m):
    if not t > 0:
        return int(np.argmax(row))
    w = weights(row, t, k, p, m)
    c = np.cumsum(w)
    return int(np.searchsorted(c / c[-1], u, side="right"))


def clear(row, u, t, k, p, m):
    """u, moved if it is near a border."""
    if not t > 0:
        return u
    c = np.cumsum(weights(row, t, k, p, m))
    c /= c[-1]
    while np.abs(c - u).min() < 1e-9:
        u = (u + 0.0137) % 1
    return u


def check(logits, u, t, k, p, m, dtype=torch.float32):
    """Every row of logits (numpy) with settings that are numbers or arrays."""
    x = torch.tensor(logits, dtype=torch.float32).to(dtype)
    rows = x.double().numpy()
    B = len(rows)
    col = [np.broadcast_to(np.asarray(c), (B,)) for c in (t, k, p, m)]
    u = np.array([clear(rows[i], u[i], *(c[i] for c in col)) for i in range(B)])
    want = [pick(rows[i], u[i], *(c[i] for c in col)) for i in range(B)]
    dev = [torch.tensor(c).cuda() if isinstance(c, np.ndarray) else c for c in (t, k, p, m)]
    got = runtime.sample_tokens(x.cuda(), torch.tensor(u).cuda(), *dev)
    assert got.dtype == torch.int32
    assert got.tolist() == want
    return got


MIXES = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (0.9, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 50, 0.95, 0.02),
         (2.0, 1, 0.5, 0.0), (0.05, 0, 0.999, 0.0), (1.0, 10 ** 6, 1e-9, 0.0), (0.0, 5, 0.5, 0.5), (-1.0, 0, 1.0, 0.0),
         (30.0, 0, 0.6, 0.9)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [1, 2, 3, 4, 5, 63, 64, 65, 1000, 1025, 4096, 12000, 32000, 65536, 151001])
def test_sample(gpu, V, dtype):
    rng = np.random.default_rng(V)
    B = 5 if V > 50000 else 12
    for mix in MIXES if V < 50000 else MIXES[:6]:
        check(2.5 * rng.standard_normal((B, V)), rng.random(B), *mix, dtype=dtype)


def test_settings_by_row(gpu):
    rng = np.random.default_rng(5)
    B, V = 64, 3001
    t = np.where(rng.random(B) < 0.2, 0.0, 0.3 + rng.random(B))
    k = rng.integers(0, 300, B) * (rng.random(B) < 0.5)
    p = np.where(rng.random(B) < 0.3, 1.0, rng.random(B))
    m = np.where(rng.random(B) < 0.5, 0.0, 0.3 * rng.random(B))
    x = 3 * rng.standard_normal((B, V))
    u = rng.random(B)
    got = check(x, u, t, k, p, m)
    # a row alone gives the same token
    rows = torch.tensor(x, dtype=torch.float32).cuda()
    dev = [torch.tensor(c).cuda() for c in (u, t, k, p, m)]
    for i in (0, 17, 63):
        alone = runtime.sample_tokens(rows[i:i + 1], dev[0][i:i + 1], float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        near = np.abs(u[i] - 0.5) < 2                # the same u unless it was moved
        if near and clear(rows[i].double().cpu().numpy(), u[i], t[i], k[i], p[i], m[i]) == u[i]:
            assert int(alone) == int(got[i])


def test_ties(gpu):
    """Equal logits: all at the k-th are kept, the nucleus takes them by index."""
    rng = np.random.default_rng(6)
    x = np.round(2 * rng.standard_normal((16, 5000)))            # about twenty values
    for mix in MIXES:
        check(x, rng.random(16), *mix)
    same = np.zeros((8, 2500))
    u = np.linspace(0.001, 0.998, 8)
    check(same, u, 1.0, 0, 1.0, 0.0)
    check(same, u, 1.0, 7, 1.0, 0.0)                             # all equal the 7-th
    check(same, u, 1.0, 0, 0.4001, 0.0)                          # the first 1001
    got = runtime.sample_tokens(torch.zeros(1, 2500).cuda(), torch.tensor([0.9999999]).cuda(), 1.0, 0, 0.4001)
    assert int(got) == 1000
    zeros = torch.tensor([[-0.0, 0.0, -1.0]]).cuda()             # one value
    assert runtime.sample_tokens(zeros, torch.tensor([0.4]).cuda(), 1.0, 1).tolist() == [0]
    assert runtime.sample_tokens(zeros, torch.tensor([0.6]).cuda(), 1.0, 1).tolist() == [1]


def test_wide_ranges(gpu):
    """Logits far apart, nearly alike, tiny and large, and masked ones."""
    rng = np.random.default_rng(7)
    B, V = 8, 3000
    base = rng.standard_normal((B, V))
    masked = np.where(rng.random((B, V)) < 0.9, -np.inf, base)
    lowest = np.where(rng.random((B, V)) < 0.9, np.finfo(np.float32).min, base)
    one = np.full((B, V), -np.inf)
    one[np.arange(B), rng.integers(0, V, B)] = -3.0
    for x in (1e-30 * base, 1e30 * base, 80 * base, 7 + 1e-6 * base, masked, lowest, one, 1e-42 * base, -base ** 2):
        for mix in MIXES:
            check(x, rng.random(B), *mix)


def test_rows_without_a_distribution(gpu):
    inf, nan = np.inf, np.nan
    x = np.array([[-inf, -inf, -inf], [1, inf, inf], [0, nan, 5], [nan, inf, nan], [-inf, 2, -inf]])
    got = runtime.sample_tokens(torch.tensor(x, dtype=torch.float32).cuda(), torch.full((5,), 0.5).cuda(), 0.8, 2, 0.9)
    assert got.tolist() == [0, 1, 1, 0, 1]
    assert runtime.sample_tokens(torch.tensor(x, dtype=torch.float32).cuda(), torch.full((5,), 0.5).cuda(),
                                 0.0).tolist() == [int(np.argmax(r)) for r in x]
    # u at and outside its range: the first and the last token that may come
    y = torch.tensor([[-inf, 1.0, 2.0, -inf]] * 4).cuda()
    u = torch.tensor([0.0, 1.0, 2.0, nan], dtype=torch.float64).cuda()
    assert runtime.sample_tokens(y, u).tolist() == [1, 2, 2, 1]
    # min-p above every weight leaves nothing
    assert runtime.sample_tokens(y[:1], u[:1], 1.0, 0, 1.0, 2.0).tolist() == [2]


def test_strides_and_types_of_settings(gpu):
    rng = np.random.default_rng(8)
    wide = torch.tensor(2 * rng.standard_normal((10, 700)), dtype=torch.float32).cuda()
    u = torch.tensor(rng.random(10)).cuda()
    for view in (wide[:, 3:503], wide[::2], wide.t()[:10], wide[:1].expand(10, 700), wide[0:10, 5:6]):
        want = runtime.sample_tokens(view.contiguous(), u[:view.shape[0]], 0.7, 30, 0.9)
        assert torch.equal(runtime.sample_tokens(view, u[:view.shape[0]], 0.7, 30, 0.9), want)
    for dt in (torch.bfloat16, torch.float16):                   # rows at odd addresses
        half = wide.to(dt)
        for view in (half[:, 1:698], half.reshape(-1)[3:3 + 9 * 701].view(9, 701), half[1::3, 7:]):
            want = runtime.sample_tokens(view.contiguous(), u[:view.shape[0]], 0.7, 30, 0.9)
            assert torch.equal(runtime.sample_tokens(view, u[:view.shape[0]], 0.7, 30, 0.9), want)
    big = torch.full((10,), (1 << 32) + 5, dtype=torch.int64, device="cuda")      # above every V: no filter
    assert torch.equal(runtime.sample_tokens(wide, u, 1.5, big), runtime.sample_tokens(wide, u, 1.5))
    f = u.float()
    assert torch.equal(runtime.sample_tokens(wide, f), runtime.sample_tokens(wide, f.double()))
    a = runtime.sample_tokens(wide, u, torch.full((10,), 0.5).cuda(), torch.full((10,), 3).cuda(), 0.75, 0.125)
    assert torch.equal(a, runtime.sample_tokens(wide, u, 0.5, 3, 0.75, 0.125))
    assert runtime.sample_tokens(wide[:0], u[:0]).shape == (0,)


def test_equals_the_host_sampler(gpu):
    """The scheduler's sampler draws one number per token; given that number the device
    picks the same token."""
    rng = np.random.default_rng(9)
    x = (2 * rng.standard_normal((40, 2000))).astype(np.float32)
    for t, k, p in ((0.8, 40, 0.95), (1.0, 0, 1.0), (0.5, 0, 0.8), (1.2, 100, 1.0)):
        for i in range(40):
            u = np.random.default_rng(i).random()
            want = sample_logits(x[i], t, p, k, np.random.default_rng(i))
            got = runtime.sample_tokens(torch.tensor(x[i:i + 1]).cuda(), torch.tensor([u]).cuda(), t, k, p)
            assert int(got) == want


def test_in_a_graph_and_on_another_stream(gpu):
    rng = np.random.default_rng(10)
    x = torch.tensor(2 * rng.standard_normal((6, 9000)), dtype=torch.float32).cuda()
    u = torch.tensor(rng.random(6)).cuda()
    want = runtime.sample_tokens(x, u, 0.8, 40, 0.95, 0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = runtime.sample_tokens(x, u, 0.8, 40, 0.95, 0.01)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = runtime.sample_tokens(x, u, 0.8, 40, 0.95, 0.01)
    for _ in range(3):
        x.copy_(2 * torch.randn_like(x))
        u.uniform_()
        graph.replay()
        want = runtime.sample_tokens(x, u, 0.8, 40, 0.95, 0.01)
        torch.cuda.synchronize()
        assert torch.equal(held, want)
