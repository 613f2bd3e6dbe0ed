"""The gradient of a decay per head against that of the same decay given to every token.

The kernels compute the same numbers either way; only where the decay's gradient goes
differs. So all other results are equal bit for bit, and the head's gradient is the sum of the
tokens', each of which was rounded to fp32 (2^-24 of it), itself rounded once. (Sums are in 64
bits, whose own roundings are below 1 % of these.) The tokens' gradients are compared with 64
bits as in test_linear_gpu.py.
"""
from __future__ import annotations

import pytest
import torch

from test_linear_edges_gpu import run
from test_linear_gpu import BF16, F16, F32, NAMES, gradients_close, inputs, ref

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])


def check(x, dtype, ref_of, cu=None):
    B, T, H, V = x["v"].shape
    gen = torch.Generator().manual_seed(9)
    dout, dsend = torch.randn(B, T, H, V, generator=gen).to(dtype).cuda(), torch.randn(x["s0"].shape, generator=gen).cuda()
    y = dict(x, g=x["g"].expand(B, T, H).contiguous())
    heads, tokens = (run([z[n] for n in NAMES], dout, dsend, cu_seqlens=cu) for z in (x, y))
    gradients_close(y, tokens[2:], dout, dsend, ref_of)
    for i, n in enumerate(("out", "send", "dq", "dk", "dv", "dg", "ds0")):
        assert n == "dg" or torch.equal(heads[i], tokens[i]), n
    got, each = heads[5].double(), tokens[5].double()
    want = each.sum((0, 1))
    room = 1.01 * 2.0 ** -24 * (each.abs().sum((0, 1)) + want.abs())
    assert got.shape == (H,) and float(room.max()) < 1e-3 * float(want.abs().max())        # can fail
    assert ((got - want).abs() <= room).all()


@TYPES
@pytest.mark.parametrize("shape", [(1, 1100, 1, 1, 128, 130), (3, 333, 1, 5, 40, 72), (2, 520, 8, 16, 64, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_sum_over_tokens(gpu, shape, dtype):
    check(inputs(*shape, dtype, seed=sum(shape), head_g=True), dtype, ref)


@TYPES
def test_sum_over_packed_tokens(gpu, dtype):
    edges = [0, 1, 300, 300, 1030]
    spans = list(zip(edges, edges[1:]))

    def packed(q, k, v, g, s0):
        res = [ref(q[:, a:e], k[:, a:e], v[:, a:e], g[:, a:e], s0[i:i + 1]) for i, (a, e) in enumerate(spans)]
        return torch.cat([r[0] for r in res], 1), torch.cat([r[1] for r in res])

    check(inputs(1, 1030, 1, 2, 20, 136, dtype, seed=8, N=len(spans), head_g=True), dtype, packed,
          torch.tensor(edges, dtype=torch.int32, device="cuda"))
