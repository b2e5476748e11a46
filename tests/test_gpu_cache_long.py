"""Cached attention over almost 2^32 tokens: the last tile's places, in each form."""
import math

import pytest
import torch

import gatgpu
from cache_cases import TYPE, words

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("precision,most", [(BF, 2), (FP, 2), (BF, 100), (BF, 200)])
def test_as_many_tokens_as_a_table_may_hold(ctx, precision, most):
    """A table of 2^28 - 1 blocks of 16 tokens, all of one page but the last, whose last token only the second row sees."""
    blocks, dim = 2 ** 28 - 1, 16
    tokens = 16 * blocks
    k, v = torch.zeros(2, 1, 16, dim, dtype=torch.uint8), torch.full((2, 1, dim, 16), 0x38, dtype=torch.uint8)
    k[1, 0, 15, 0] = 0x78   # 2^8, in the queries' only column
    v[1, 0, :, 15] = 0x40   # 2, else 1
    k, v, scales = k.cuda(), v.cuda(), torch.ones(4, device="cuda")
    table = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    table[-1] = 1
    cache = gatgpu.Cache(pages=2, page=16, kv_heads=1, dim=dim, k=k.data_ptr(), v=v.data_ptr(), k_scale=scales.data_ptr(), v_scale=scales.data_ptr())
    q = torch.zeros(2, dim, dtype=TYPE[precision], device="cuda")
    q[:, 0] = 1.0
    out, lse = torch.full_like(q, 7.0), torch.full((2, 1), 7.0, device="cuda")
    begin, lens = words([0, 2]), words([tokens])
    scale = 32 * math.log(2.0) / 256  # the last token's score: 32, as a power of 2
    io = gatgpu.CacheAttentionIO(precision=precision, heads=1, scale=scale, rows=2, requests=1, most=most, blocks=blocks, table_stride=blocks, q=q.data_ptr(),
                                 q_stride=dim, q_begin=begin.data_ptr(), k_len=lens.data_ptr(), table=table.data_ptr(), out=out.data_ptr(), out_stride=dim,
                                 lse=lse.data_ptr())
    work = torch.empty(ctx.cache_attention_workspace(cache, io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.cache_attention(cache, io, work.data_ptr(), work.numel())
    ctx.synchronize()
    # Row 0: 2^32 - 17 tokens of score 0 and value 1; row 1: one more, of weight 2^32 and value 2.  The score is off by at most
    # 32 * 2^-22, sums of equal weights by nothing up to 2^24 of them and by 2^-24 each time that waves and pieces are joined.
    w = 2.0 ** 32
    want = [(1.0, math.log(w - 17)), ((w - 17 + 2 * w) / (2 * w - 17), math.log(2 * w - 17))]
    step = 2.0 ** -8 if precision == BF else 0.0
    for i, (x, l) in enumerate(want):
        assert bool(((out[i].double() - x).abs() <= x * (step + 2.0 ** -15)).all()), out[i]
        assert abs(float(lse[i]) - l) <= 2.0 ** -15, float(lse[i])
