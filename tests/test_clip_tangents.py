"""The gradients' norm and their clipping have no forward-mode derivative: a tensor with a
tangent is refused, where a scaled value beside its old tangent would be wrong."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from sunnynet_amd import runtime


def test_tangents_are_refused():
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(NotImplementedError, match="grad_norm"):
            runtime.grad_norm([x, dual])
        for grads, out in (([x, dual], None), (iter([dual]), None), ([dual], [torch.empty(3)]), ([x], [dual])):
            with pytest.raises(NotImplementedError, match="clip_grad_norm"):
                runtime.clip_grad_norm(grads, 1.0, out=out)
        for call in (runtime.grad_norm, lambda g: runtime.clip_grad_norm(g, 1.0)):      # as outside of a dual level
            with pytest.raises(ValueError, match="one GPU"):
                call([x])
            with pytest.raises(ValueError, match="leave out"):
                call([None])
