"""Segment attention at the ends of its values' ranges, against the plain computation in 64 bits (attention_cases.py)."""
import pytest

import gatgpu
from attention_cases import Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", [(300, 300, 4, 2), (1, 600, 4, 2), (1, 9000, 8, 8), (384, 384, 32, 32)])
@pytest.mark.parametrize("train", [False, True])
def test_large_values_under_capped_scores(ctx, precision, q_len, k_len, heads, kv_heads, train):
    """Scores near their cap, whose weights without a reference are 2^86, and values of 2^60: the sums pass FP32, the
    outputs do not."""
    p = Problem([q_len], [k_len], heads, kv_heads, 32, precision, cap=60.0, scale=20.0, seed=k_len)
    p.v *= 2.0 ** 60
    p.dout *= 2.0 ** -60
    p.check(p.run(ctx, train), train)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", [(300, 300, 4, 2), (1, 600, 4, 2), (1, 9000, 8, 8), (384, 384, 32, 32)])
def test_small_values_under_scores_near_minus_the_cap(ctx, precision, q_len, k_len, heads, kv_heads):
    """The same from below: all weights are 2^-86, and values of 2^-60 with them are none of FP32's normal numbers."""
    p = Problem([q_len], [k_len], heads, kv_heads, 32, precision, cap=60.0, scale=20.0, seed=k_len + 1)
    p.q.abs_()
    p.k.abs_().neg_()
    p.v *= 2.0 ** -60
    p.check(p.run(ctx, train=False), train=False)


def test_some_rows_near_minus_the_cap(ctx):
    """Beside ordinary rows of the same tiles, under a prefix mask that leaves some rows nothing."""
    p = Problem([310], [300], 4, 2, 32, BF, mask=gatgpu.MASK_PREFIX, cap=60.0, seed=5)
    p.k[:, 0, 0] = 9.0
    p.q[100:120, :2, 0] = -400.0
    p.v *= 2.0 ** -60
    p.check(p.run(ctx, train=False), train=False)
