"""Norms of queries and keys whose squares leave FP32's normal numbers, on the GPU against the plain computation in 64 bits."""
import math

import pytest
import torch

import gatgpu
from test_gpu_rotate import HALVES, NEIGHBOURS, Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def sized(p, size):
    """Rows of `size`, but for every third, which stays as it is."""
    keep = torch.arange(p.x.shape[0]) % 3 == 2
    p.x = torch.where(keep.view(-1, 1), p.x, (p.x.double() * size).to(p.x.dtype))
    return p


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim,rot,pairs", [(64, 64, HALVES), (64, 20, HALVES), (40, 40, NEIGHBOURS), (8, 8, NEIGHBOURS), (256, 128, HALVES), (128, 0, HALVES)])
@pytest.mark.parametrize("size", [1e-15, 1e-18, 1e-20, 1e-22, 1e-25, 1e-30, 1e-34])
def test_small_rows_without_eps(ctx, precision, dim, rot, pairs, size):
    """Mean squares among FP32's subnormal numbers and below them: x and y differ by a factor only, and dx is large."""
    p = sized(Problem(25, 6, 2, dim, precision, rot=rot, pairs=pairs, seed=dim + rot, gap=1), size)
    p.eps = 0.0
    p.dy = (p.dy.double() * min(1.0, size * 1e30)).to(p.dy.dtype)  # (so that dx is an FP32 number)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("size,eps", [(1e-20, 1e-39), (1e-20, 1e-44), (1e-22, 1e-38), (1e-10, 1e-30), (1e-17, 1e-34)])
def test_small_rows_with_a_small_eps(ctx, precision, size, eps):
    p = sized(Problem(25, 3, 1, 64, precision, seed=3), size)
    p.eps = float(torch.tensor(eps, dtype=torch.float32))
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim,rot,pairs", [(64, 64, HALVES), (64, 20, HALVES), (40, 40, NEIGHBOURS), (256, 128, HALVES)])
@pytest.mark.parametrize("eps", [0.0, 1e-5, 1e30])
@pytest.mark.parametrize("size", [1e15, 1e18, 1e19, 1e25, 2e37])
def test_large_rows(ctx, precision, dim, rot, pairs, size, eps):
    """Squares beyond FP32's range."""
    p = sized(Problem(25, 6, 2, dim, precision, rot=rot, pairs=pairs, seed=dim + rot, gap=1), size)
    assert bool(torch.isfinite(p.x.float()).all())
    p.eps = float(torch.tensor(eps, dtype=torch.float32))
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_rows_of_zeros_nan_and_infinity_stay_by_themselves(ctx, precision):
    """Without eps a row of zeros is 0 / 0; none of them changes another row or head."""
    made = [Problem(20, 3, 2, 64, precision, seed=10) for _ in range(2)]
    x = made[0].x
    x[4, 64:128] = 0.0              # query head 1 of row 4
    x[5, 3 * 64 + 1] = math.inf     # key head 0 of row 5
    x[6, 4 * 64 + 7] = math.nan     # key head 1 of row 6
    for p in made:
        p.eps = 0.0
    got, want = (p.run(ctx) for p in made)
    same = torch.ones(x.shape, dtype=torch.bool)
    same[4, 64:128] = same[5, 192:256] = same[6, 256:320] = False
    for n in ("y", "dx"):
        a, b = got[n].cpu(), want[n].cpu()
        assert torch.equal(a[same], b[same])
    y = got["y"].cpu()
    assert bool(torch.isnan(y[4, 64:128]).all()) and bool(torch.isnan(y[6, 256:320]).all()) and not bool(torch.isfinite(y[5, 192:256]).all())
