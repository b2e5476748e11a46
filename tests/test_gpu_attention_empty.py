"""Batches without query rows, without key rows and without either: torch gives their empty arrays the address 0."""
import math

import pytest
import torch

import gatgpu
from attention_cases import Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
NONE, LINEAR, TABLE = gatgpu.BIAS_NONE, gatgpu.BIAS_LINEAR, gatgpu.BIAS_TABLE
QUERIES, KEYS = ("q", "out", "lse", "rest", "dout", "dq"), ("k", "v", "dk", "dv")


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def run(ctx, p, without):
    """Forward and backward with a null pointer and stride for each array of `without`."""
    with p.plan(ctx) as plan:
        out, io = p.buffers()
        for name in without:
            setattr(io, name, None)
            if name not in ("lse", "rest"):
                setattr(io, name + "_stride", 0)
        ws = torch.empty(max(1, plan.workspace_bytes(), plan.workspace_bytes(backward=True)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        plan.forward(io, ws.data_ptr(), ws.numel())
        plan.backward(io, ws.data_ptr(), ws.numel())
        ctx.synchronize()
    return out


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("bias,buckets", [(NONE, 0), (LINEAR, 0), (TABLE, 5)])
def test_no_rows_at_all(ctx, precision, bias, buckets):
    for lens in ([], [0], [0, 0, 0]):
        p = Problem(lens, lens, 4, 2, 32, precision, bias=bias, buckets=buckets)
        out = run(ctx, p, QUERIES + KEYS)
        if bias == TABLE:
            assert bool((out["dbias"] == 0).all())


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("mask", [gatgpu.MASK_FULL, gatgpu.MASK_PREFIX])
@pytest.mark.parametrize("bias,buckets", [(NONE, 0), (LINEAR, 0), (TABLE, 5)])
@pytest.mark.parametrize("lens", [[5], [40, 0, 300], [2000]])
def test_queries_without_keys(ctx, precision, mask, bias, buckets, lens):
    p = Problem(lens, [0] * len(lens), 4, 2, 64, precision, mask=mask, bias=bias, buckets=buckets)
    out = run(ctx, p, KEYS)
    assert bool((out["out"] == 0).all()) and bool((out["lse"] == -math.inf).all()) and bool((out["dq"] == 0).all())
    if bias == TABLE:
        assert bool((out["dbias"] == 0).all())


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("mask", [gatgpu.MASK_FULL, gatgpu.MASK_PREFIX])
@pytest.mark.parametrize("bias,buckets", [(NONE, 0), (LINEAR, 0), (TABLE, 5)])
@pytest.mark.parametrize("lens", [[5], [40, 0, 300], [2000]])
def test_keys_without_queries(ctx, precision, mask, bias, buckets, lens):
    p = Problem([0] * len(lens), lens, 4, 2, 64, precision, mask=mask, bias=bias, buckets=buckets)
    out = run(ctx, p, QUERIES)
    assert bool((out["dk"] == 0).all()) and bool((out["dv"] == 0).all())
    if bias == TABLE:
        assert bool((out["dbias"] == 0).all())


def test_arrays_with_rows_are_still_refused(ctx):
    p = Problem([3, 0], [0, 4], 4, 2, 32, BF)
    for name in QUERIES + KEYS:
        if name != "rest":
            with pytest.raises(gatgpu.GatGpuError) as err:
                run(ctx, p, (name,))
            assert err.value.code == gatgpu.EINVAL
