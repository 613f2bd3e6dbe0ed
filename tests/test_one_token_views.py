"""Views of one token out of a large (token, batch, head, column) array: their token axis has
a stride beyond the kernels' range, which nothing uses."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime
from sunnynet_amd.runtime.delta import MAX_STRIDE, _rows


def far(t):
    """t, of one token, with that axis' stride out of range."""
    s = t.stride()
    return t.as_strided(t.shape, (s[0], MAX_STRIDE + 8, *s[2:]), t.storage_offset())


def test_rows_have_strides_in_range():
    t = torch.randn(2, 1, 3, 4)
    for x in (far(t), far(t.transpose(0, 2)), far(torch.randn(2, 1, 3, 8)[..., ::2]), far(torch.randn(2, 1, 3, 8)[..., 4:])):
        assert x.stride(1) >= MAX_STRIDE
        y = _rows(x)
        assert all(s < MAX_STRIDE for s in y.stride()) and y.stride(-1) == 1 and torch.equal(x, y)
    assert _rows(t) is t and _rows(far(t)).data_ptr() == t.data_ptr()        # no copy


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear_attention", "gated_delta"])
def test_calls_take_them(gpu, name):
    B, H, K, V = 2, 3, 8, 16
    call = getattr(runtime, name)
    q, k, v = (torch.randn(B, 1, H, n, device=gpu) for n in (K, K, V))
    rest = [-torch.rand(B, 1, H, device=gpu)] * (1 if name == "linear_attention" else 2)
    s0 = torch.randn(B, H, K, V, device=gpu)
    want = call(q, k, v, *rest, s0)
    got = call(far(q), far(k), far(v), *rest, s0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = []
    for wide in (lambda t: t, far):
        leaf = [t.clone().requires_grad_() for t in (q, k, v)]
        out, send = call(*(wide(t) for t in leaf), *rest, s0)
        grads.append((out, send, *torch.autograd.grad(out.sum() + send.square().sum(), leaf)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
