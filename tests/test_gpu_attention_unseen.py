"""Single NaN and infinities in keys, queries, values and gradients of pairs that are not seen: they reach nothing.

Every test takes the reference of clean inputs, plants the bad elements and holds what they must not reach
against that reference, within the bounds of attention_cases.py.  One element, not a row, is bad, so that
products stay infinities of either sign; a mask by position hides the score, not the operand.
"""
import math

import pytest
import torch

import gatgpu
from attention_cases import HIDDEN, Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
VALUES = [math.nan, math.inf, -math.inf]
# Backward kernels of one, two and four waves that hold all keys; of one and of four waves a block; of ranges
LENGTHS = [(20, 32), (50, 64), (100, 32), (132, 64), (384, 32), (1100, 32)]
CAPS = [0.0, 3.0]


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def close(got, ref, rows, name):
    """got[name] at `rows` (an index of the outputs' rows and heads) within its bound."""
    val, tol = ref
    have, want, off = got[name].double()[rows], val[name][rows], tol[name][rows]
    assert bool((torch.isfinite(have) == torch.isfinite(want)).all()), f"{name}: not finite"
    fine = torch.isfinite(want)
    assert bool(((have - want).abs() <= off + 1e-30)[fine].all()), name


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("n,dim", LENGTHS)
@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("cap", CAPS)
def test_a_key_behind_the_rows(ctx, precision, n, dim, value, cap):
    """Causal mask: the last key is bad and only the last query sees it."""
    p = Problem([n], [n], 4, 2, dim, precision, mask=gatgpu.MASK_PREFIX, cap=cap, seed=n)
    ref = p.reference()
    p.k[n - 1, 0, 3] = value
    got = p.run(ctx)
    for name in ("out", "lse", "dq"):
        close(got, ref, slice(0, n - 1), name)
        close(got, ref, (slice(None), slice(2, 4)), name)  # the heads of the other key/value head
    for name in ("dk", "dv"):
        close(got, ref, (slice(None), 1), name)
    if math.isnan(value):
        assert bool(torch.isnan(got["out"][n - 1, :2]).all()) and bool(torch.isnan(got["dq"][n - 1, :2]).all())
        assert bool(torch.isnan(got["dk"][:, 0]).all()) and bool(torch.isnan(got["dv"][:, 0]).all())


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("n,dim", LENGTHS)
@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("cap", CAPS)
def test_queries_that_see_nothing(ctx, precision, n, dim, value, cap):
    """Causal mask, nine queries more than keys: the first nine see none."""
    p = Problem([n + 9], [n], 4, 2, dim, precision, mask=gatgpu.MASK_PREFIX, cap=cap, seed=n + 1)
    ref = p.reference()
    p.q[4, 0, 3], p.q[8, 3, 0], p.dout[5, 1, 2] = value, value, value
    got = p.run(ctx)
    for name in ref[0]:
        close(got, ref, slice(None), name)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("n,dim", LENGTHS)
@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1)])
def test_pairs_hidden_by_the_table(ctx, precision, n, dim, value, cap, heads, kv_heads):
    """A key and a query without any visible pair, and a key whose table entry is -infinity."""
    p = Problem([n], [n], heads, kv_heads, dim, precision, bias=gatgpu.BIAS_TABLE, buckets=5, cap=cap, seed=n + 2)
    d, i, j, k = p.distances(0), n // 2, n - 2, n // 3
    p.table[:, 4] = -math.inf
    d[d >= 4] = HIDDEN
    d[:, k] = 4
    d[i], d[:, j] = HIDDEN, HIDDEN
    ref = p.reference()
    p.k[j, 0, 3], p.v[j, 0, 1], p.k[k, 0, 0], p.q[i, 0, 5], p.dout[i, 0, 7] = (value,) * 5
    got = p.run(ctx)
    for name in ref[0]:
        close(got, ref, slice(None), name)
