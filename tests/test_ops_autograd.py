"""What the operators owe autograd besides gradients, where nothing has to run on a GPU."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from sunnynet_amd import runtime

NAMES = ("q", "k", "v", "g", "beta", "s0")


def delta_args(step):
    lead = (2,) if step else (2, 20)
    return [torch.rand(*lead, *s) for s in ((1, 8), (1, 8), (2, 6), (2,), (2,))] + [torch.rand(2, 2, 8, 6)]


def calls():
    """(name, call of a list of tensors, the tensors)."""
    yield "gated_delta", lambda a: runtime.gated_delta(*a), delta_args(False)
    yield "delta_step", lambda a: runtime.delta_step(*a), delta_args(True)
    yield "layer_norm", lambda a: runtime.layer_norm(*a), [torch.rand(3, 8), torch.rand(8), torch.rand(8)]


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_tangents_are_refused_not_dropped(grad):
    """A dual tensor has no requires_grad; whichever argument is one, the call is refused."""
    for name, call, args in calls():
        for i in range(len(args)):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                duals = list(args)
                duals[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match=name):
                    call(duals)
                with pytest.raises(ValueError, match="one GPU"):       # inside the level, without a tangent
                    call(args)
        with pytest.raises(NotImplementedError, match=name):
            torch.func.jvp(lambda x: call([x, *args[1:]]), (args[0],), (args[0],))


def test_a_tracked_send_is_refused():
    """Writing a tensor that autograd tracks would leave its history wrong."""
    args = delta_args(True)
    with pytest.raises(RuntimeError, match="gated_delta"):
        runtime.delta_step(*args, send=torch.zeros_like(args[5]).requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="one GPU"):
        runtime.delta_step(*args, send=torch.zeros_like(args[5]).requires_grad_())
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="delta_step"):
        runtime.delta_step(*args, send=forward_ad.make_dual(torch.zeros_like(args[5]), torch.ones_like(args[5])))
