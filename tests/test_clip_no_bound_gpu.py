"""A bound without end clips nothing, whatever the norm; only a norm of NaN makes all NaN."""
from __future__ import annotations

import math

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [0.5, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_no_bound(gpu, dtype, value):
    xs = [torch.randn(n, device=gpu).to(dtype) for n in (300, 9000)]
    xs[1][77] = value
    kept = [x.clone() for x in xs]
    ys = [torch.empty_like(x) for x in xs]
    norms = runtime.clip_grad_norm(xs, math.inf, out=ys), runtime.clip_grad_norm(xs, math.inf)
    for norm in norms:
        assert torch.isnan(norm) if math.isnan(value) else float(norm) == float(runtime.grad_norm(kept))
    for x, y, z in zip(kept, ys, xs):
        if math.isnan(value):
            assert y.isnan().all() and z.isnan().all()
        else:
            assert torch.equal(x, y) and torch.equal(x, z)
