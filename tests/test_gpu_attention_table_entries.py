"""Where a table entry begins to hide its pairs (gatgpu.h): from -1e6 down, and not above."""
import math

import numpy as np
import pytest
import torch

import gatgpu
from attention_cases import Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
HIDES = np.float32(-1e6)
COUNTS = np.nextafter(HIDES, np.float32(0))


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", [(20, 20, 2, 2), (60, 60, 2, 1), (100, 100, 4, 4), (200, 200, 2, 2), (1, 600, 8, 8), (2, 9000, 4, 4)])
def test_entries_at_the_border(ctx, precision, q_len, k_len, heads, kv_heads):
    """Rows with nothing else: hidden by the one, a softmax among equals by the other; beside other keys neither weighs."""
    p = Problem([q_len], [k_len], heads, kv_heads, 32, precision, bias=gatgpu.BIAS_TABLE, buckets=4, hidden=0.0, seed=k_len)
    p.table[:, 1], p.table[:, 2:] = float(HIDES), float(COUNTS)
    d = p.distances(0)
    d[:, ::2], d[:, 1::2] = 1, 2
    d[q_len // 2:, :5] = 0
    d[q_len // 3] = 1
    d[0] = 2 if q_len > 1 else 1
    got = p.run(ctx)
    p.check(got)
    if q_len > 1:
        assert bool((got["lse"][0] < -9e5).all()) and bool(torch.isfinite(got["lse"][0]).all())
        # equal biases of such a size leave a score steps of 1/8: weights within 2^(1/8) of their softmax
        a = p.v.double().abs().amax()
        assert float(got["out"][0].double().abs().max()) <= float(a) * 1.1 and float(got["out"][0].double().abs().max()) > 0
    at = q_len // 3 if q_len // 3 else 0
    if q_len == 1 or at:
        assert bool((got["out"][at] == 0).all()) and bool((got["lse"][at] == -math.inf).all())
