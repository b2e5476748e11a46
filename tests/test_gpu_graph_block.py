"""A graph transformer's block, as a user runs it: a GAT layer over the edges with its norm, attention
among all nodes of each graph with a table of biases by distance, the residual's norm, and back.

The calls follow each other on the context's stream without a pause; then each one is held against
its formula in 64 bits on the arrays that it was really given, within that formula's own bound.
"""
import numpy as np
import pytest
import torch

import gatgpu
from attention_cases import Problem
from gatgpu import inputs
from test_gpu_norm import Norm, model_norms, plain_norm

pytestmark = pytest.mark.gpu

FP, BF = gatgpu.FP32, gatgpu.BF16
LENS = [9, 60, 31, 1, 130, 64, 300, 5]
HEADS, DIM = 8, 32


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


class Block:
    """Arrays of one block of `precision` rows; nodes of all graphs packed one behind the other."""

    def __init__(self, ctx, precision):
        n, w = sum(LENS), HEADS * DIM
        self.att = Problem(LENS, LENS, HEADS, HEADS, DIM, precision, bias=gatgpu.BIAS_TABLE, buckets=12, seed=41, packed=False)
        self.norm = Norm(n, w, precision, residual=True, elu=False, seed=42)
        self.out, self.io = self.att.buffers()
        self.norm.x = self.out["out"].view(n, w)  # the attention's rows ...
        self.norm_out, self.norm_io = self.norm.arrays()
        self.att.dout = self.norm_out["dx"].view(n, HEADS, DIM)  # ... and their gradient
        self.io.dout, self.io.dout_stride = self.norm_out["dx"].data_ptr(), w
        self.plan = self.att.plan(ctx)
        self.need = max(1, self.plan.workspace_bytes(), self.plan.workspace_bytes(backward=True))
        self.ws = torch.empty(self.need, dtype=torch.uint8, device="cuda")
        self.norm_ws = torch.empty(ctx.norm_workspace(n, w), dtype=torch.uint8, device="cuda")

    def set_rows(self, hidden):
        """Hidden rows [n][256] are queries, keys, values and residual."""
        rows = hidden.to(self.att.t).contiguous()
        self.norm.residual = rows
        self.norm_io.residual, self.norm_io.residual_stride = rows.data_ptr(), rows.stride(0)
        self.att.q = self.att.k = self.att.v = rows.view(-1, HEADS, DIM)
        for x in "qkv":
            setattr(self.io, x, rows.data_ptr())
            setattr(self.io, x + "_stride", rows.stride(0))

    def run(self, ctx):
        self.plan.forward(self.io, self.ws.data_ptr(), self.need)
        ctx.norm_forward(self.norm_io)
        ctx.norm_backward(self.norm_io, self.norm_ws.data_ptr(), self.norm_ws.numel())
        self.plan.backward(self.io, self.ws.data_ptr(), self.need)

    def check(self):
        self.att.check(self.out)
        self.norm.check(self.norm_out)


@pytest.mark.parametrize("precision", [FP, BF])
def test_block_forward_and_backward(ctx, precision):
    n = sum(LENS)
    row, col = inputs.powerlaw_graph(n, 6 * n, 60, 43)
    x = inputs.normal((n, 48), 44)
    layer = inputs.glorot_param(48, HEADS, DIM, 45)
    gamma, beta = model_norms([layer], 46)[0]
    ctx.set_graph(row, col)
    ctx.set_layer(0, layer)
    ctx.layer_forward(0, precision, gatgpu.TRANSFORM_FIRST, False, input=x)
    raw = ctx.stage(0, "out")
    ctx.set_norm(0, gamma, beta)
    try:
        block = Block(ctx, precision)
        xd = torch.from_numpy(x).cuda()
        hidden = torch.full((n, HEADS * DIM), 7.0, device="cuda")
        block.set_rows(hidden)
        torch.cuda.synchronize()
        ctx.layer_forward_static(0, precision, True, xd.data_ptr(), hidden.data_ptr())
        if precision == FP:  # (in FP32 the layer's output is the block's input as it stands)
            for a in "qkv":
                setattr(block.io, a, hidden.data_ptr())
            block.norm_io.residual = hidden.data_ptr()
            block.run(ctx)
            ctx.synchronize()
            block.set_rows(hidden)
        else:
            ctx.synchronize()
            block.set_rows(hidden)
            torch.cuda.synchronize()
            block.run(ctx)
            ctx.synchronize()
        # 256 columns: 300 u of a normalised value of at most 16 times gamma
        assert np.abs(hidden.cpu().numpy() - plain_norm(raw, gamma, beta, 1e-5, True)).max() < 300 * 2.0 ** -24 * 16 * 2.5
        block.check()
        block.plan.close()
    finally:
        ctx.set_norm(0, None, None)


@pytest.mark.parametrize("precision", [FP, BF])
def test_block_replays(ctx, precision):
    """Captured once, replayed on other rows, with eager work of the same context between."""
    block, other = Block(ctx, precision), Block(ctx, precision)
    g = torch.Generator(device="cuda").manual_seed(47)
    n, w = sum(LENS), HEADS * DIM
    block.set_rows(torch.randn(n, w, generator=g, device="cuda"))
    torch.cuda.synchronize()
    block.run(ctx)
    ctx.synchronize()
    stream = torch.cuda.ExternalStream(ctx.stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        block.run(ctx)
    for _ in range(3):
        rows = torch.randn(n, w, generator=g, device="cuda")
        block.norm.residual.copy_(rows)
        other.set_rows(rows)
        for out in (block.out, block.norm_out):
            for a in out.values():
                a.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        other.run(ctx)
        ctx.synchronize()
        for have, want in ((block.out, other.out), (block.norm_out, other.norm_out)):
            for name in have:
                if name != "rest":
                    assert torch.equal(have[name], want[name]), name
    block.check()
    block.plan.close()
    other.plan.close()
