"""The operators inside other graphs, on the GPU."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import runtime

pytestmark = pytest.mark.gpu


def step_args(dev):
    gen = torch.Generator(dev).manual_seed(1)

    def rn(*s):
        return torch.randn(*s, generator=gen, device=dev)

    return [rn(2, 1, 8), rn(2, 1, 8), rn(2, 2, 6), -rn(2, 2).abs(), torch.sigmoid(rn(2, 2))], rn(2, 2, 8, 6)


@pytest.mark.parametrize("apart", [False, True], ids=["in_place", "send"])
def test_a_graph_that_saved_the_state_refuses_a_stepped_one(gpu, apart):
    """w's gradient needs the state that the forward read: once delta_step has written over it,
    the backward pass is an error and no wrong number."""
    args, s = step_args(gpu)
    kept = torch.zeros_like(s) if apart else s
    w = torch.ones_like(s).requires_grad_()
    read = (kept * w).sum()
    runtime.delta_step(*args, s, send=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        read.backward()
    again = (kept * w).sum()                # the new state, read after the step
    want = kept.clone()
    again.backward()
    assert torch.equal(w.grad, want)


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_the_plain_recurrence_counts_as_modifying_its_state(gpu, where):
    """The step of the plain recurrence writes s in place behind a raw pointer."""
    a, b, s = (torch.rand(2, 8, device=where) for _ in range(3))
    w = torch.ones(2, 8, device=where, requires_grad=True)
    read = (s * w).sum()
    runtime.step(a, b, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        read.backward()


def test_a_send_that_overlaps_the_state_is_refused(gpu):
    """Heads are read and written in no order, so only the same place or another one will do."""
    args, s = step_args(gpu)
    both = torch.zeros(2, *s.shape, device=gpu)
    both[0] = s
    flat = both.view(-1)
    with pytest.raises(ValueError, match="apart"):
        runtime.delta_step(*args, both[0], send=flat[1:1 + s.numel()].view(s.shape))
    same = both[0].clone()
    out = runtime.delta_step(*args, both[0], send=both[1])
    assert torch.equal(runtime.delta_step(*args, both[0], send=flat[:s.numel()].view(s.shape)), out)
    assert torch.equal(both[0], both[1]) and not torch.equal(both[0], same)
