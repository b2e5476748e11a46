"""Plans near the end of what one launch takes."""
import pytest
import torch

import gatgpu
from attention_cases import Problem

pytestmark = pytest.mark.gpu


def test_blocks_of_four_waves_that_a_launch_does_not_take():
    """66000 segments of 385 rows, 64 heads: 13 waves each are 3.5e9 threads, four blocks of four waves 4.3e9."""
    n, q_len, k_len, heads, dim = 66000, 385, 129, 64, 8
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.empty(n * q_len, heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    k, v = (torch.empty(n * k_len, heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    out = torch.full_like(q, 7.0)
    with gatgpu.Context(0) as ctx, gatgpu.Attention(ctx, [q_len] * n, [k_len] * n, heads=heads, dim=dim) as plan:
        ws = torch.empty(max(1, plan.workspace_bytes()), dtype=torch.uint8, device="cuda")
        io = gatgpu.AttentionIO(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_stride=heads * dim,
                                k_stride=heads * dim, v_stride=heads * dim, out_stride=heads * dim)
        torch.cuda.synchronize()
        plan.forward(io, ws.data_ptr(), ws.numel())
        ctx.synchronize()
    for s in (0, 1, n // 2, n - 2, n - 1):
        p = Problem([q_len], [k_len], heads, heads, dim, seed=2, packed=False)
        p.q, p.k, p.v = (x[s * m:(s + 1) * m] for x, m in ((q, q_len), (k, k_len), (v, k_len)))
        val, tol = p.reference(train=False)
        have = out[s * q_len:(s + 1) * q_len].double()
        assert bool(((have - val["out"]).abs() <= tol["out"]).all()), s
    assert not bool((out.view(n, -1)[:, -1] == 7.0).any())  # every segment's last element is an output
    del q, k, v, out, ws
    torch.cuda.empty_cache()
