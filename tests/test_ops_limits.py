"""Ends of the operators' documented ranges, where nothing has to run on a GPU."""
from __future__ import annotations

import pytest
import torch

from sunnynet_amd import _native, runtime
from sunnynet_amd.runtime import delta

P = 4096        # stands for a device pointer: a refused call reads no array


def pack(dims, cu=0, dtype=0, chunks=P, states=P):
    return delta._ARGS.pack(P, P, P, P, P, 0, cu, *([1] * 9), *dims, dtype, 1.0, chunks, states)


@pytest.mark.parametrize("i", range(7), ids=["B", "T", "N", "Hk", "H", "K", "V"])
@pytest.mark.parametrize("value", [0, -1, 1 << 62])
def test_workspaces_of_sizes_out_of_range_are_empty(i, value):
    """The size queries answer 0 for what the calls refuse, whatever the numbers are."""
    L = _native.lib()
    good = [2, 50, 2, 2, 4, 8, 6]
    sizes = L.snhip_op_delta_chunk_floats, L.snhip_op_delta_state_floats, L.snhip_op_delta_bwd_floats
    assert all(f(pack(good)) > 0 for f in sizes)
    dims = list(good)
    dims[i] = value
    assert [f(pack(dims)) for f in sizes] == [0, 0, 0]
    assert L.snhip_op_delta_fwd_dev(pack(dims), P, P, None) == -1
    assert [f(pack(good, dtype=3)) for f in sizes] == [0, 0, 0]
    assert [f(None) for f in sizes] == [0, 0, 0]


def test_chunks_that_no_launch_holds_are_refused():
    """Up to 512 threads a chunk, and fewer than 2^32 in a grid's dimension: 2^23 chunks of 32
    tokens are too many for the calls with workspaces."""
    L = _native.lib()
    sizes = L.snhip_op_delta_chunk_floats, L.snhip_op_delta_state_floats, L.snhip_op_delta_bwd_floats
    grads = delta._GRAD.pack(*[P] * 9)
    for dims, cu in (((1, 1 << 28, 1, 1, 1, 8, 8), 0), ((4, 1 << 26, 4, 1, 1, 8, 8), 0),
                     ((1, (1 << 28) - 32, 1, 1, 1, 8, 8), P)):
        assert L.snhip_op_delta_fwd_dev(pack(dims, cu), P, P, None) == -1
        assert L.snhip_op_delta_bwd_dev(pack(dims, cu), grads, None) == -1
        assert [f(pack(dims, cu)) for f in sizes] == [0, 0, 0]
    assert all(f(pack((1, (1 << 28) - 32, 1, 1, 1, 8, 8))) > 0 for f in sizes)
    meta = [torch.empty(1, 1 << 28, 1, n, device="meta") for n in (8, 8, 8)]
    gates = [torch.empty(1, 1 << 28, 1, device="meta") for _ in range(2)]
    with pytest.raises(ValueError, match="chunks"):
        runtime.gated_delta(*meta, *gates)
