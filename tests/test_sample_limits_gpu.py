"""Sampling at the ends of its ranges: more rows than a launch holds, rows at the documented
limits, and settings far from 1."""
from __future__ import annotations

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
