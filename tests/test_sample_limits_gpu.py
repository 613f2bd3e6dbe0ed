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
