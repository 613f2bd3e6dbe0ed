"""Sampling at the ends of its ranges: more rows than a launch holds, rows at the documented
limits, and settings far from 1."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_holds(gpu):
    """2^23 rows of 512 threads each are 2^32 threads, one more than a grid's dimension takes.
    Rows at the ends and around the launches' borders are those of their own calls."""
    B, V = (1 << 23) + 5, 3
    gen = torch.Generator(gpu).manual_seed(2)
    x = torch.empty(B, V, dtype=torch.float16, device=gpu).normal_(generator=gen)
    f64 = dict(dtype=torch.float64, device=gpu, generator=gen)
    u, t, p, m = (torch.rand(B, **f64) for _ in range(4))
    k = torch.randint(0, 4, (B,), dtype=torch.int32, device=gpu, generator=gen)
    t, m = t + 0.2, 0.5 * m
    got = runtime.sample_tokens(x, u, t, k, p, m)
    assert bool(((got >= 0) & (got < V)).all())
    for at in (0, (1 << 22) - 50, B - 100):
        part = slice(at, at + 100)
        assert torch.equal(runtime.sample_tokens(x[part], u[part], t[part], k[part], p[part], m[part]), got[part])
    greedy = runtime.sample_tokens(x, u, 0.0)
    assert torch.equal(greedy.long(), x.float().argmax(1))


def test_whether_u_chose_the_token(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[0.0, 1, 2, 3, -inf], [nan, 1, 2, 3, 4], [1, inf, 0, 0, 0], [-inf] * 5, [1, 2, 3, 4, 5]], device=gpu)
    u = torch.full((5,), 0.3, device=gpu)
    t = torch.tensor([1.0, 1, 1, 1, 0], device=gpu)
    for more in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.9, 0.0), (2, 0.9, 0.1)):
        both = runtime.sample_tokens(x, u, t, *more, drew=True)
        assert both.shape == (2, 5) and both[1].tolist() == [1, 0, 0, 0, 0]
        assert torch.equal(both[0], runtime.sample_tokens(x, u, t, *more))
        assert both[0, 1:].tolist() == [0, 1, 0, 4]
    for k in (0, 2):                       # min-p above every weight leaves nothing
        assert runtime.sample_tokens(x[:1], u[:1], 1.0, k, 1.0, 2.0, drew=True).tolist() == [[3], [0]]
    assert runtime.sample_tokens(x[:0], u[:0], drew=True).shape == (2, 0)


def test_top_k_by_row_of_other_types(gpu):
    """Numbers that 32 bits do not hold filter as they are: none below 1, none from V on."""
    gen = torch.Generator(gpu).manual_seed(4)
    x = torch.randn(6, 900, device=gpu, generator=gen)
    u = torch.rand(6, dtype=torch.float64, device=gpu, generator=gen)
    none, five = runtime.sample_tokens(x, u, 1.5), runtime.sample_tokens(x, u, 1.5, 5)
    assert not torch.equal(none, five)
    far = [-(1 << 32) + 5, (1 << 32) + 5, -(1 << 62), 1 << 62, -1, 0]
    assert torch.equal(runtime.sample_tokens(x, u, 1.5, torch.tensor(far, device=gpu)), none)
    for dt in (torch.float32, torch.float64):
        far = torch.tensor([-1e30, 1e30, float("inf"), -float("inf"), float("nan"), 0.0], dtype=dt, device=gpu)
        assert torch.equal(runtime.sample_tokens(x, u, 1.5, far), none)
    for dt in (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.float16, torch.float64):
        k = torch.full((6,), 5, dtype=dt, device=gpu)
        assert torch.equal(runtime.sample_tokens(x, u, 1.5, k), five)
    assert torch.equal(runtime.sample_tokens(x, u, 1.5, 10 ** 30), none)
    assert torch.equal(runtime.sample_tokens(x, u, 1.5, -10 ** 30), none)


def pick(row, u, t, k, p, m):
    """The definition for one row of float64 (temperature > 0)."""
    z = row / t
    w = np.exp(z - z.max())
    if 0 < k < z.size:
        w[z < np.sort(z)[-k]] = 0.0
    if 0 < p < 1:
        order = np.argsort(-z, kind="stable")
        ws = w[order]
        cut = np.cumsum(ws) - ws > p * ws.sum()
        cut[0] = False
        w[order[cut]] = 0.0
    w[w < m] = 0.0
    c = np.cumsum(w) / w.sum()
    return int(np.searchsorted(c, u, side="right")), np.abs(c - u).min()


def test_logits_further_apart_than_fp32_reaches(gpu):
    """Differences of two finite logits that are infinite in fp32, at a temperature that makes
    them ordinary. Random numbers nearer than 1e-9 to a border are left out."""
    rng = np.random.default_rng(5)
    x = torch.tensor(rng.uniform(-3.4e38, 3.4e38, (40, 700)), dtype=torch.float32)
    rows, tested = x.double().numpy(), 0
    for t in (1e38, 4e37, 3e39):
        for k, p, m in ((0, 1.0, 0.0), (600, 1.0, 0.0), (0, 0.97, 0.0), (650, 0.9, 0.01), (120, 1.0, 0.0)):
            u = rng.random(40)
            got = runtime.sample_tokens(x.to(gpu), torch.tensor(u).to(gpu), t, k, p, m).tolist()
            for i in range(40):
                want, near = pick(rows[i], u[i], t, k, p, m)
                if near > 1e-9:
                    assert got[i] == want, (t, k, p, m, i)
                    tested += 1
    assert tested > 590


LONG = [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (0.9, 0, 0.9, 0.02), (1.2, 700, 0.8, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [8193, 12000, 65537])
def test_many_long_rows(gpu, V, dtype):
    """More than 256 rows of more than 8192 logits: rows of 8 waves, against the definition and
    against calls of fewer rows, which have 16."""
    rng = np.random.default_rng(V)
    for B in (257, 512):
        x = torch.tensor(2.5 * rng.standard_normal((B, V)), dtype=torch.float32).to(dtype)
        rows, u, dev = x[:6].double().numpy(), rng.random(B), x.to(gpu)
        for mix in LONG:
            near = [pick(rows[i], u[i], *mix) for i in range(6)]
            got = runtime.sample_tokens(dev, torch.tensor(u).to(gpu), *mix)
            for i, (want, gap) in enumerate(near):
                if gap > V * 2.0 ** -45:               # the weights' rounding at this V: below 2^-46 each
                    assert int(got[i]) == want, (mix, i)
            half = [runtime.sample_tokens(dev[s], torch.tensor(u[s]).to(gpu), *mix)
                    for s in (slice(0, 200), slice(200, 400), slice(400, B)) if s.start < B]
            assert torch.equal(torch.cat(half), got)


@pytest.mark.parametrize("V", [(1 << 20) - 1, 1 << 20])
def test_the_longest_rows(gpu, V):
    """Weights are whole multiples of 2^-42 of the largest, so shares are off by less than
    V 2^-43, and with the total's own rounding less than V 2^-42: random numbers and nuclei
    nearer than that to a border are moved."""
    rng = np.random.default_rng(V)
    x = torch.tensor(6 * rng.standard_normal(V), dtype=torch.float32)
    row, near = x.double().numpy(), V * 2.0 ** -42
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.8, 5000, 1.0, 0.0), (0.9, 0, 0.6, 0.0), (1.0, 200, 0.9, 1e-3)):
        if p < 1:
            z = np.sort(row)[::-1] / t
            w = np.exp(z - z[0])
            if k:
                w = w[:k]
            edge = np.cumsum(w) / w.sum()
            while np.abs(edge - p).min() < near:
                p += 1e-4
        u, want = [], []
        while len(u) < 300:
            c = rng.random()
            if len(u) < 3:
                tok, gap = pick(row, c, t, k, p, m)
                if gap < near:
                    continue
                want.append(tok)
            u.append(c)
        u = torch.tensor(u, dtype=torch.float64).to(gpu)
        few = runtime.sample_tokens(x.to(gpu)[None].expand(3, V), u[:3], t, k, p, m)
        many = runtime.sample_tokens(x.to(gpu)[None].expand(300, V), u, t, k, p, m)
        assert few.tolist() == want and torch.equal(many[:3], few)
        assert torch.equal(many[-3:], runtime.sample_tokens(x.to(gpu)[None].expand(3, V), u[-3:], t, k, p, m))
