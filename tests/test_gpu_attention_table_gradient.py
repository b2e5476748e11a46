"""The table's gradient of bf16 rows is FP32: delta = dout.out keeps FP32's digits, where ds = p (dp - delta) cancels.

Queries are 0, so that scores are the table's entries, and dout is 1 in column 0, so that dp is v's column 0 and delta is out's,
each exactly: what is left of the gradient's error is that of out with its rest.  u is 2^-24.
"""
import math

import pytest
import torch

import gatgpu
from attention_cases import Problem

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def problem(q_len, k_len, heads, kv_heads, buckets):
    p = Problem([q_len], [k_len], heads, kv_heads, 32, gatgpu.BF16, bias=gatgpu.BIAS_TABLE, buckets=buckets, hidden=0.0, seed=k_len)
    for x in (p.q, p.v, p.dout):
        x.zero_()
    p.dout[..., 0] = 1
    p.table.zero_()
    p.distances(0)[:] = 0
    return p


# Forward kernels: of short segments (heads that the short backward pass does not take), of one and of four waves a block, with
# keys cut among waves, with ranges that a launch joins
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads", [(20, 30, 3, 1), (70, 30, 6, 2), (150, 150, 2, 2), (300, 300, 32, 32), (384, 384, 64, 64),
                                                        (1, 600, 8, 8), (2, 9000, 8, 4), (1, 300, 40, 40)])
def test_equal_weights(ctx, q_len, k_len, heads, kv_heads):
    """One bucket: the gradient is 0.  Values of 1 and 1 + 2^-7, as many of each as leave out farthest from bf16 and a bf16 rest."""
    p = problem(q_len, k_len, heads, kv_heads, 1)
    # (with one rest of bf16, out would be off by up to 2^-17, 128 u)
    r = torch.arange(1, k_len // 2, dtype=torch.float64) / k_len / 128
    m = 1 + int((r - r.to(torch.bfloat16).double()).abs().argmax())
    assert abs(m / k_len / 128 - float(torch.tensor(m / k_len / 128).to(torch.bfloat16))) > 40 * U
    p.v[..., 0] = 1
    p.v[:m, :, 0] += 2.0 ** -7
    got = p.run(ctx)
    # Sums of v are exact.  out: the sum of the weights (32 of them and more a range, scales of joins: 4 u), its reciprocal, the product;
    # rest 2 u.  p is off by 2 |lse2| u + 6 u relative, |dp - delta| at most 2^-7; the sums of ds, of at most 2^-7 a row, run in at most
    # k_len / 2 + 64 additions a term.
    lse2 = math.log2(k_len)
    bound = q_len * (12 * U + 2.0 ** -7 * (2 * lse2 + 6 + k_len / 2 + 64) * U)
    assert float(got["dbias"].abs().max()) <= bound


@pytest.mark.parametrize("q_len,heads,kv_heads", [(64, 16, 16), (32, 24, 8), (1, 48, 48), (384, 16, 16)])
def test_unequal_weights(ctx, q_len, heads, kv_heads):
    """130 keys, of which eight have value 1 and weigh 2^7 to 2^7.9 times the others, a weight that no two bf16 hold."""
    p = problem(q_len, 130, heads, kv_heads, 2)
    heavy = slice(70, 78)
    p.distances(0)[:, heavy] = 1
    p.v[heavy, :, 0] = 1
    p.table[:, 1] = torch.linspace(7.0, 7.9, heads, device="cuda") * math.log(2)
    got = p.run(ctx)
    t = p.table[:, 1].double()
    w = 8 * torch.exp(t) / (8 * torch.exp(t) + 122)
    assert float((got["lse"].double() - torch.log(8 * torch.exp(t) + 122)).abs().max()) < 1e-5
    # dbias of the heavy: each query's sum of p (1 - w) over them, w (1 - w); of the others minus that.
    # The heavy weight is off by 16 u relative (its score to 8 u, half of that a rounding of either entry, and the exponential), out by
    # 16 u (1 - w) of that, 8 u of the sum of weights, 8 u of sums, joins and the product, and 2 u of rest, relative; p in the
    # backward pass by 40 u, the sums of ds by 80 u.
    off = w * (18 * U * w + (1 - w) * (16 + 40 + 80) * U)
    assert bool(((got["dbias"][:, 1].double() - q_len * w * (1 - w)).abs() <= q_len * off).all())
