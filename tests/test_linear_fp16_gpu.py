"""Packed calls of linear attention in fp16 against 64 bits, as test_linear_gpu.py and
test_linear_edges_gpu.py have them for the other types."""
from __future__ import annotations

import pytest

import test_linear_edges_gpu as edge_tests
import test_linear_gpu as tests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("edges", [[0, 5, 5, 70, 900], [0, 0, 0, 1], [3, 67, 131, 700, 1000], [0, 64, 128, 1024]],
                         ids=str)
def test_packed(gpu, edges):
    tests.test_packed(gpu, edges, tests.F16)


def test_packed_with_a_decay_per_head(gpu):
    edge_tests.test_packed_with_a_decay_per_head(gpu, tests.F16)
