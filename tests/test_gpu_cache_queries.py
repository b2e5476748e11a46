"""Cached attention of queries that are infinite or near FP32's ends, in each form."""
import math

import pytest
import torch

import gatgpu
from cache_cases import Serving

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
FORMS = [(FP, 16), (FP, 40), (FP, 400), (BF, 16), (BF, 40), (BF, 400)]
forms = pytest.mark.parametrize("precision,most", FORMS)


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@forms
def test_scores_of_minus_infinity(ctx, precision, most):
    """A query of -infinity in a column where every key is positive sees no finite score; beside it rows of finite ones."""
    p = Serving([100, 70], [9, 16], 4, 2, 32, 16, precision, seed=90)
    p.host.k[..., 3] = 0x30   # 0.5
    p.q[2, 1, 3], p.q[20, 0, 3] = -math.inf, -math.inf
    d = p.run(ctx, most=most)
    p.check(d)
    out, lse = d["out"].cpu()[:, :128].view(-1, 4, 32), d["lse"].cpu()
    assert lse[2, 1] == -math.inf and lse[20, 0] == -math.inf and bool((out[2, 1] == 0).all()) and bool((out[20, 0] == 0).all())


@pytest.mark.parametrize("most", [16, 40, 400])
def test_the_largest_queries(ctx, most):
    """FP32 queries up to the largest number, which bf16 does not hold, over keys that are as small."""
    p = Serving([100, 70], [9, 16], 4, 2, 32, 16, FP, seed=91)
    p.host.k_scale[:] = 2.0 ** -64
    top = float(torch.finfo(torch.float32).max)
    p.q = p.q.sign() * top * (1 - 2.0 ** -20 * p.q.abs())
    p.q[0], p.q[1, :, 5:] = top, 0.0
    p.host.k[..., 1:] = 0   # (one product a score: its sum stays within FP32)
    p.host.k[..., 0] &= 0x87   # less than 2^-6
    p.scale = 2.0 ** -50
    p.check(p.run(ctx, most=most))
