"""Refusals of linear attention, the embedding and clipping that need no GPU: the Python
entry points check shapes, types and devices before any device work, and the C calls
return SNHIP_E_INVAL for arguments outside their ranges."""
from __future__ import annotations

from array import array

import pytest
import torch

from sunnynet_amd import _native, runtime
from sunnynet_amd.runtime import clip, linear

B, T, Hk, H, K, V = 2, 5, 2, 4, 8, 6
P = 4096        # stands for a device pointer: a refused call reads no array


def good():
    return {"q": torch.zeros(B, T, Hk, K), "k": torch.zeros(B, T, Hk, K), "v": torch.zeros(B, T, H, V),
            "g": torch.zeros(B, T, H), "s0": torch.zeros(B, H, K, V)}


@pytest.mark.parametrize("bad, what", [
    ({"q": torch.zeros(B, T, Hk, K + 1)}, "shape"),
    ({"q": torch.zeros(T, Hk, K)}, "shape"),
    ({"v": torch.zeros(B, T + 1, H, V)}, "shape"),
    ({"g": torch.zeros(B, T, H + 1)}, "shape"),
    ({"g": torch.zeros(T, H)}, "shape"),
    ({"g": torch.zeros(Hk)}, "shape"),
    ({"g": torch.zeros(())}, "shape"),
    ({"v": torch.zeros(B, T, 3, V), "g": torch.zeros(B, T, 3)}, "share"),
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
    ({"g": torch.zeros(H)}, "one GPU"),
])
def test_linear_refuses(bad, what):
    with pytest.raises(ValueError, match=what):
        runtime.linear_attention(**{**good(), **bad})


def test_linear_step_refuses():
    x = {n: t[:, 0] if n != "s0" else t for n, t in good().items()}
    for bad, what in (({"q": torch.zeros(B, 1, Hk, K)}, "shape"), ({"g": torch.zeros(B, H, 1)}, "shape"),
                      ({"s0": torch.zeros(B, H, V, K)}, "s0"), ({}, "one GPU")):
        y = {**x, **bad}
        with pytest.raises(ValueError, match=what):
            runtime.linear_step(y["q"], y["k"], y["v"], y["g"], y["s0"])
    x["v"].requires_grad_()
    with pytest.raises(RuntimeError, match="linear_attention"):
        runtime.linear_step(*x.values())
    with torch.no_grad(), pytest.raises(ValueError, match="one GPU"):
        runtime.linear_step(*x.values())


def test_embed_refuses():
    table, ids = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for args, what in (((torch.zeros(5), ids), "R, D"), ((torch.zeros(0, 8), ids), "R, D"),
                       ((torch.zeros(5, 0), ids), "R, D"), ((torch.zeros(1, (1 << 20) + 1), ids), "R, D"),
                       ((table.double(), ids), "float32"), ((table, ids.short()), "int32"),
                       ((table, ids.float()), "int32"), ((table, ids), "one GPU")):
        with pytest.raises(ValueError, match=what):
            runtime.embed(*args)
    with pytest.raises(ValueError, match="contiguous"):
        runtime.embed_bwd(torch.zeros(8, 3).t(), ids, 5)
    with pytest.raises(ValueError, match="shape"):
        runtime.embed_bwd(torch.zeros(4, 8), ids, 5)


def test_clip_refuses():
    x = [torch.zeros(5), torch.zeros(3)]
    for args, what in ((([],), "no gradients"), ((x,), "one GPU"), (([None],), "leave out")):
        with pytest.raises(ValueError, match=what):
            runtime.grad_norm(*args)
        with pytest.raises(ValueError, match=what):
            runtime.clip_grad_norm(*args, 1.0)
    for bound in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="negative"):
            runtime.clip_grad_norm(x, bound)
    with pytest.raises(RuntimeError, match="leaf"):
        runtime.clip_grad_norm([torch.zeros(3, requires_grad=True)], 1.0)


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        x = good()
        x["k"] = forward_ad.make_dual(x["k"], torch.ones_like(x["k"]))
        with pytest.raises(NotImplementedError):
            runtime.linear_attention(**x)
        table = forward_ad.make_dual(torch.zeros(5, 8), torch.ones(5, 8))
        with pytest.raises(NotImplementedError):
            runtime.embed(table, torch.zeros(3, dtype=torch.int64))


def pack(q=P, g=P, cu=0, stride=1, dims=(B, T, B, Hk, H, K, V), dtype=0, head_g=0, parts=0):
    return linear._ARGS.pack(q, P, P, g, 0, cu, *([1, stride, 1] * 3), *dims, dtype, head_g, 1.0, parts)


def test_linear_c_calls_refuse():
    L = _native.lib()
    grads = linear._GRAD.pack(*[P] * 9)
    for b in [dict(q=0), dict(g=0), dict(dims=(0, T, 0, Hk, H, K, V)), dict(dims=(B, 0, B, Hk, H, K, V)),
              dict(dims=(B, T, B + 1, Hk, H, K, V)), dict(dims=(B, T, B, 3, H, K, V)),
              dict(dims=(B, T, B, Hk, H, 129, V)), dict(dims=(B, T, B, Hk, H, K, 4097)),
              dict(dims=(B, T, B, Hk, H, 0, V)), dict(dims=(2, 1 << 29, 2, Hk, H, K, V)),
              dict(dims=(1, 1 << 30, 1, Hk, H, K, V)), dict(dims=(B, T, 3, Hk, H, K, V), cu=P),
              dict(dims=(65536, 1, 65536, Hk, H, K, V)), dict(dims=(1, 1, 1, 1, 65535, 128, 256)), dict(dtype=3),
              dict(dtype=-1), dict(stride=-1), dict(stride=1 << 24), dict(parts=P + 4)]:
        a = pack(**b)
        assert L.snhip_op_linear_fwd_dev(a, P, P, None) == -1, b
        assert L.snhip_op_linear_step_dev(a, P, P, None) == -1, b
        assert L.snhip_op_linear_bwd_dev(a, grads, None) == -1, b
    assert L.snhip_op_linear_fwd_dev(pack(), None, P, None) == -1
    assert L.snhip_op_linear_fwd_dev(None, P, P, None) == -1
    assert L.snhip_op_linear_step_dev(pack(), P, None, None) == -1
    assert L.snhip_op_linear_step_dev(pack(cu=P, dims=(1, T, 3, Hk, H, K, V)), P, P, None) == -1
    long = (1, 1 << 20, 1, Hk, H, K, V)                     # needs its workspace
    assert L.snhip_op_linear_parts_floats(pack(dims=long)) > 0
    assert L.snhip_op_linear_fwd_dev(pack(dims=long), P, P, None) == -1
    assert L.snhip_op_linear_bwd_dev(pack(dims=long), grads, None) == -1
    for i in (0, 2, 3, 4, 5, 6, 8):            # every array but dsend and ds0 (send where dsend is)
        g = [P] * 9
        g[i] = 0
        assert L.snhip_op_linear_bwd_dev(pack(), linear._GRAD.pack(*g), None) == -1, i
    assert L.snhip_op_linear_bwd_dev(pack(), linear._GRAD.pack(*[P] * 8, P + 4), None) == -1


@pytest.mark.parametrize("i", range(7), ids=["B", "T", "N", "Hk", "H", "K", "V"])
@pytest.mark.parametrize("value", [0, -1, 1 << 62])
def test_linear_workspaces_of_sizes_out_of_range_are_empty(i, value):
    L = _native.lib()
    dims = [1, 1 << 20, 1, 2, 4, 8, 6]
    sizes = L.snhip_op_linear_parts_floats, L.snhip_op_linear_bwd_floats
    assert all(f(pack(dims=dims)) > 0 for f in sizes)
    dims[i] = value
    assert [f(pack(dims=dims)) for f in sizes] == [0, 0]
    assert [f(pack(dtype=3)) for f in sizes] == [0, 0] and [f(None) for f in sizes] == [0, 0]


def test_embed_c_calls_refuse():
    L = _native.lib()
    fwd, bwd, size = L.snhip_op_embed_fwd_dev, L.snhip_op_embed_bwd_dev, L.snhip_op_embed_bwd_bytes
    for t, i, y in ((0, P, P), (P, 0, P), (P, P, 0)):
        assert fwd(t, i, 1, y, 3, 5, 8, 1.0, 0, None) == -1
        assert bwd(t, i, 1, y, P, 3, 5, 8, 1.0, 0, None) == -1
    assert bwd(P, P, 1, P, None, 3, 5, 8, 1.0, 0, None) == -1 and bwd(P, P, 1, P, P + 4, 3, 5, 8, 1.0, 0, None) == -1
    for n, R, D, kind in ((0, 5, 8, 0), (1 << 31, 5, 8, 0), (3, 0, 8, 0), (3, (1 << 28) + 1, 8, 0), (3, 5, 0, 0),
                          (3, 5, (1 << 20) + 1, 0), (3, 5, 8, 3), (3, 5, 8, -1)):
        assert fwd(P, P, 1, P, n, R, D, 1.0, kind, None) == -1
        assert bwd(P, P, 1, P, P, n, R, D, 1.0, kind, None) == -1
        assert size(n, R, D, kind) == 0
    assert size(3, 5, 8, 0) > 0


def test_clip_c_calls_refuse():
    """Overlaps, sizes and types; nothing of these reaches the device."""
    L = _native.lib()

    def run(x, y, n, kinds, count=None, norm=P, ws=P):
        a = [array("Q", x), array("Q", y) if y is not None else None, array("q", n), array("i", kinds)]
        return L.snhip_op_clip_dev(clip._ARGS.pack(*(0 if t is None else t.buffer_info()[0] for t in a),
                                                   len(n) if count is None else count, 1.0, ws), norm, None)

    one, two = 1 << 20, (1 << 20) + 4000
    assert run([one], [one], [10], [0], norm=None) == -1 and run([one], [one], [10], [0], ws=0) == -1
    assert run([one], [one], [10], [3]) == -1 and run([one], [one], [10], [-1]) == -1
    assert run([one], [one], [-1], [0]) == -1 and run([one], [one], [1 << 36], [0]) == -1
    assert run([one], [one], [10], [0], count=-1) == -1 and run([one], [one], [10], [0], count=1 << 20) == -1
    assert run([0], [one], [10], [0]) == -1 and run([one], [0], [10], [0]) == -1
    assert run([one, one], [one, one], [10, 10], [0, 0]) == -1                 # one gradient twice
    assert run([one, two], [one, two], [1001, 10], [0, 0]) == -1               # one inside the other
    assert run([one, two], [two, one], [10, 10], [0, 0]) == -1                 # changed places
    assert run([one], [one + 16], [10], [0]) == -1                             # a part of itself
    assert run([one, two], [two + 100, two + 100], [10, 10], [0, 0]) == -1     # one place for both
    assert L.snhip_op_clip_doubles(-1) == 0 and L.snhip_op_clip_doubles(1 << 20) == 0
    assert L.snhip_op_clip_doubles(0) > 0 and L.snhip_op_clip_doubles(300) == 3 * L.snhip_op_clip_doubles(1)
