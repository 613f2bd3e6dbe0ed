"""Refusals of the delta rule, layer norm and sampling that need no GPU: the Python
entry points check shapes, types and devices before any device work, and the C calls
return SNHIP_E_INVAL for arguments outside their ranges."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import _native, runtime
from sunnynet_amd.runtime import delta, sample

B, T, Hk, H, K, V = 2, 5, 2, 4, 8, 6


def good():
    return {"q": torch.zeros(B, T, Hk, K), "k": torch.zeros(B, T, Hk, K), "v": torch.zeros(B, T, H, V),
            "g": torch.zeros(B, T, H), "beta": torch.zeros(B, T, H), "s0": torch.zeros(B, H, K, V)}


@pytest.mark.parametrize("bad, what", [
    ({"q": torch.zeros(B, T, Hk, K + 1)}, "shape"),
    ({"q": torch.zeros(T, Hk, K)}, "shape"),
    ({"v": torch.zeros(B, T + 1, H, V)}, "shape"),
    ({"g": torch.zeros(B, T, H + 1)}, "shape"),
    ({"beta": torch.zeros(B, T)}, "shape"),
    ({"v": torch.zeros(B, T, 3, V), "g": torch.zeros(B, T, 3), "beta": torch.zeros(B, T, 3)}, "share"),
    ({"q": torch.zeros(B, T, Hk, 129), "k": torch.zeros(B, T, Hk, 129)}, "head sizes"),
    ({"q": torch.zeros(B, T, Hk, 0), "k": torch.zeros(B, T, Hk, 0)}, "head sizes"),
    ({"v": torch.zeros(B, T, H, 4097)}, "head sizes"),
    ({"q": torch.zeros(B, T, Hk, K).half()}, "all three"),
    ({n: torch.zeros(B, T, Hk, K).double() for n in "qk"}, "all three"),
    ({"g": torch.zeros(B, T, H).bfloat16()}, "float32"),
    ({"s0": torch.zeros(B, H, V, K)}, "s0"),
    ({"s0": torch.zeros(B, H, K, V).half()}, "s0"),
    ({"cu_seqlens": torch.zeros(3, dtype=torch.int32)}, "B must be 1"),
    ({"cu_seqlens": torch.zeros(3)}, "int32"),
    ({"cu_seqlens": torch.zeros(1, dtype=torch.int32)}, "int32"),
    ({}, "one GPU"),
])
def test_delta_refuses(bad, what):
    with pytest.raises(ValueError, match=what):
        runtime.gated_delta(**{**good(), **bad})


def test_delta_step_refuses():
    x = {n: t[:, 0] if n != "s0" else t for n, t in good().items()}
    for bad, what in (({"q": torch.zeros(B, 1, Hk, K)}, "shape"), ({"g": torch.zeros(B, H, 1)}, "shape"),
                      ({"s0": torch.zeros(B, H, V, K)}, "s0"), ({}, "one GPU")):
        y = {**x, **bad}
        with pytest.raises(ValueError, match=what):
            runtime.delta_step(y["q"], y["k"], y["v"], y["g"], y["beta"], y["s0"])


def test_delta_step_refuses_a_tape():
    x = {n: t[:, 0] if n != "s0" else t for n, t in good().items()}
    x["v"].requires_grad_()
    with pytest.raises(RuntimeError, match="gated_delta"):
        runtime.delta_step(x["q"], x["k"], x["v"], x["g"], x["beta"], x["s0"])
    with torch.no_grad(), pytest.raises(ValueError, match="one GPU"):
        runtime.delta_step(x["q"], x["k"], x["v"], x["g"], x["beta"], x["s0"])


def test_norm_refuses():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for args, what in (((x, torch.ones(7)), "length D"), ((x, w.half()), "float32"), ((x.double(),), "float32"),
                       ((torch.zeros(2, 16385),), "D from 1"), ((torch.zeros(2, 0),), "D from 1"),
                       ((x, w, torch.zeros(9)), "length D"), ((x, w), "one GPU")):
        with pytest.raises(ValueError, match=what):
            runtime.layer_norm(*args)
    with pytest.raises(ValueError, match="contiguous"):
        runtime.norm_fwd(torch.zeros(8, 4).t())


def test_sample_refuses():
    x, u = torch.zeros(3, 8), torch.zeros(3)
    for args, what in (((torch.zeros(8), u), "B, V"), ((torch.zeros(3, 0), u), "V from 1"),
                       ((torch.zeros(1, sample.MAX_V + 1), u[:1]), "V from 1"), ((x.double(), u), "float32"),
                       ((x, u), "device tensors")):
        with pytest.raises(ValueError, match=what):
            runtime.sample_tokens(*args)


P = 4096        # stands for a device pointer: a refused call reads no array


def _delta(chunks=P, states=0, q=P, cu=0, dims=(B, T, B, Hk, H, K, V), dtype=0):
    return delta._ARGS.pack(q, P, P, P, P, 0, cu, *([1] * 9), *dims, dtype, 1.0, chunks, states)


def test_c_calls_refuse():
    L = _native.lib()
    bad = [dict(q=0), dict(dims=(0, T, 0, Hk, H, K, V)), dict(dims=(B, 0, B, Hk, H, K, V)),
           dict(dims=(B, T, B + 1, Hk, H, K, V)), dict(dims=(B, T, B, 3, H, K, V)),
           dict(dims=(B, T, B, Hk, H, 129, V)), dict(dims=(B, T, B, Hk, H, K, 4097)),
           dict(dims=(B, T, B, Hk, H, 0, V)), dict(dims=(2, 1 << 29, 2, Hk, H, K, V)), dict(dims=(1, 1 << 30, 1, Hk, H, K, V)),
           dict(dims=(B, T, 3, Hk, H, K, V), cu=P), dict(dims=(65536, 1, 65536, Hk, H, K, V)), dict(dtype=3),
           dict(dtype=-1)]
    grads = delta._GRAD.pack(*[P] * 9)
    for b in bad:
        a = _delta(states=P, **b)
        assert L.snhip_op_delta_fwd_dev(a, P, P, None) == -1, b
        assert L.snhip_op_delta_step_dev(a, P, P, None) == -1, b
        assert L.snhip_op_delta_bwd_dev(a, grads, None) == -1, b
    assert L.snhip_op_delta_fwd_dev(_delta(), None, P, None) == -1
    assert L.snhip_op_delta_fwd_dev(_delta(chunks=P + 4), P, P, None) == -1          # workspaces 16-byte aligned
    assert L.snhip_op_delta_fwd_dev(_delta(states=P + 8), P, P, None) == -1
    assert L.snhip_op_delta_bwd_dev(_delta(states=P), delta._GRAD.pack(*[P] * 8, P + 4), None) == -1
    wide = delta._ARGS.pack(P, P, P, P, P, 0, 0, *([1, 1 << 24, 1] * 3), B, T, B, Hk, H, K, V, 0, 1.0, P, 0)
    back = delta._ARGS.pack(P, P, P, P, P, 0, 0, *([1, -1, 1] * 3), B, T, B, Hk, H, K, V, 0, 1.0, P, 0)
    assert L.snhip_op_delta_fwd_dev(wide, P, P, None) == -1 and L.snhip_op_delta_fwd_dev(back, P, P, None) == -1
    assert L.snhip_op_delta_fwd_dev(None, P, P, None) == -1
    assert L.snhip_op_delta_step_dev(_delta(), P, None, None) == -1
    # without a workspace only short calls
    assert L.snhip_op_delta_fwd_dev(_delta(chunks=0, dims=(B, 17, B, Hk, H, K, V)), P, P, None) == -1
    assert L.snhip_op_delta_fwd_dev(_delta(chunks=0, states=P), P, P, None) == -1
    assert L.snhip_op_delta_fwd_dev(_delta(chunks=0, cu=P, dims=(1, T, 3, Hk, H, K, V)), P, P, None) == -1
    for i in (0, 2, 3, 4, 5, 6, 8):            # every array but dsend and ds0
        g = [P] * 9
        g[i] = 0
        assert L.snhip_op_delta_bwd_dev(_delta(states=P), delta._GRAD.pack(*g), None) == -1
    assert L.snhip_op_delta_bwd_dev(_delta(), grads, None) == -1          # no states
    n = L.snhip_op_norm_fwd_dev
    assert n(None, P, P, P, P, P, 4, 8, 1e-5, 0, None) == -1
    assert n(P, P, P, P, P, None, 4, 8, 1e-5, 0, None) == -1
    assert n(P, P, P, P, P, P, 0, 8, 1e-5, 0, None) == -1
    assert n(P, P, P, P, P, P, 4, 16385, 1e-5, 0, None) == -1
    assert n(P, P, P, P, P, P, 4, 8, 1e-5, 3, None) == -1
    n = L.snhip_op_norm_bwd_dev
    assert n(P, P, P, None, P, P, P, P, P, 4, 8, 0, None) == -1
    assert n(P, P, P, P, P, P, P, None, None, 4, 8, 0, None) == -1
    assert n(P, P, P, P, P, P, P, P, P, 1 << 31, 8, 0, None) == -1
    s = lambda **k: sample._ARGS.pack(k.get("x", P), k.get("u", P), 0, 0, 0, 0, 1.0, 1.0, 0.0, 0,  # noqa: E731
                                      k.get("B", 2), k.get("V", 8), k.get("stride", 8), k.get("dtype", 0))
    for b in (dict(x=0), dict(u=0), dict(B=0), dict(V=0), dict(V=(1 << 20) + 1), dict(stride=-8), dict(dtype=3)):
        assert L.snhip_op_sample_dev(s(**b), P, None) == -1, b
    assert L.snhip_op_sample_dev(s(), None, None) == -1


def test_workspace_sizes():
    L = _native.lib()
    size = [L.snhip_op_delta_chunk_floats(_delta(dims=(B, t, B, Hk, H, K, V))) for t in (1, 32, 33)]
    assert size[0] == size[1] and size[2] == 2 * size[1]
    # packed sequences: a chunk more for each of them at most
    assert L.snhip_op_delta_chunk_floats(_delta(cu=P, dims=(1, 100, 7, Hk, H, K, V))) == (100 // 32 + 7) * size[0] // B
    assert L.snhip_op_delta_state_floats(_delta(dims=(1, 32, 1, 1, 1, 65, 17))) == (128 + 32) * 32
    assert L.snhip_op_norm_bwd_floats(0, 8) == 0 and L.snhip_op_norm_bwd_floats(1, 8) == 2 * 8
    assert L.snhip_op_norm_bwd_floats(10 ** 6, 8) == L.snhip_op_norm_bwd_floats(10 ** 7, 8) > 0
