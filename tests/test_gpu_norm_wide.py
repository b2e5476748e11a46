"""Rows so wide that the sums of their weights' gradients pass one grid dimension."""
import pytest
import torch

import gatgpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("rows", [1, 2])
def test_gradients_of_very_many_columns(rows):
    """2^26 + 41 columns: 32 of the sums' 2 W columns a block of 1024 threads pass 2^32."""
    w = (1 << 26) + 41
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.empty(rows, w, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = (torch.empty(rows, device="cuda") for _ in range(2))
    dgamma, dbeta = (torch.full((w,), 7.0, device="cuda") for _ in range(2))
    with gatgpu.Context(0) as ctx:
        ws = torch.empty(ctx.norm_workspace(rows, w), dtype=torch.uint8, device="cuda")
        io = gatgpu.NormIO(precision=gatgpu.BF16, rows=rows, width=w, eps=1e-5, x=x.data_ptr(), x_stride=w, y=y.data_ptr(), y_stride=w,
                           mean=mean.data_ptr(), rstd=rstd.data_ptr(), dy=dy.data_ptr(), dy_stride=w, dx=dx.data_ptr(), dx_stride=w,
                           dgamma=dgamma.data_ptr(), dbeta=dbeta.data_ptr())
        torch.cuda.synchronize()
        ctx.norm_forward(io)
        ctx.norm_backward(io, ws.data_ptr(), ws.numel())
        ctx.synchronize()
    n = (x.double() - mean.double().view(-1, 1)) * rstd.double().view(-1, 1)
    # n by two rounded operations, its product by one, and the rows' sum by one
    size = (n * dy.double()).abs().sum(0)
    assert float(((dgamma.double() - (n * dy.double()).sum(0)).abs() - 4 * U * size).max()) <= 0
    assert float(((dbeta.double() - dy.double().sum(0)).abs() - U * dy.double().abs().sum(0)).max()) <= 0
    # each of 1024 threads adds 2^16 values of a mean of 0.8, then 1024 sums: at most 2^16 + 16 roundings a sum
    assert float((mean.double() - x.double().mean(1)).abs().max()) <= 65552 * U * 0.9
    del x, dy, y, dx, dgamma, dbeta, ws, n, size
    torch.cuda.empty_cache()
