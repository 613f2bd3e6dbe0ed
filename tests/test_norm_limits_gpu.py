"""Layer norm over more rows than one launch holds."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_holds(gpu):
    """2^26 rows of 64 threads each are 2^32 threads, one more than a grid's dimension takes.
    Rows at the ends and around the launches' borders have the bits of their own calls."""
    R, D = (1 << 26) + 5, 2
    gen = torch.Generator(gpu).manual_seed(1)
    x = torch.empty(R, D, dtype=torch.float16, device=gpu).normal_(generator=gen)
    w, b = torch.tensor([1.25, 0.5], device=gpu), torch.tensor([0.0, 3.0], device=gpu)
    y, mean, rstd = runtime.norm_fwd(x, w, b, keep=True)
    for at in (0, (1 << 23) - 50, (1 << 25) - 50, R - 100):
        part = slice(at, at + 100)
        for a, c in zip(runtime.norm_fwd(x[part], w, b, keep=True), (y, mean, rstd)):
            assert torch.equal(a, c[part])
    assert bool((mean - x.float().mean(1)).abs().max() <= 2.0 ** -22 * x.float().abs().max())
    assert bool(rstd.isfinite().all())
