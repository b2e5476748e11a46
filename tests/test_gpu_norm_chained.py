"""Norms of the model's layers in the chained forward: every layer's stored output is the one that the layer gives alone."""
import numpy as np
import pytest

import gatgpu
from gatgpu import inputs
from test_gpu_norm import model_norms

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("normed", [(0,), (1,), (2,), (0, 1), (0, 1, 2)])
@pytest.mark.parametrize("fuse", [0, 2])
def test_outputs_of_a_chain(ctx, precision, normed, fuse):
    row, col = inputs.powerlaw_graph(2500, 30000, 500, 15)
    x = inputs.normal((2500, 100), 16)
    model = inputs.glorot_model(100, 8, 32, 47, 17)
    norms = model_norms(model, 18)
    ctx.set_graph(row, col)
    ctx.set_model(model)
    ctx.set_input(x)
    ctx.set_option(gatgpu.OPT_FUSE_NEXT_PROJECTION, fuse)
    try:
        for l in normed:
            ctx.set_norm(l, *norms[l], 1e-5)
        h, alone = x, []
        for l in range(3):
            ctx.layer_forward(l, precision, gatgpu.TRANSFORM_FIRST, l < 2, input=h)
            h = ctx.stage(l, "out")
            alone.append(h)
        logits = ctx.model_forward(precision, gatgpu.TRANSFORM_FIRST)[0]
        assert np.array_equal(logits, alone[2]) and np.array_equal(ctx.stage(2, "out"), alone[2])
        for l in (0, 1):
            if l in normed:  # (others may hand their rows to the next projection without storing them)
                assert ctx.has_stage(l, "out")
            if ctx.has_stage(l, "out"):
                assert np.array_equal(ctx.stage(l, "out"), alone[l]), l
    finally:
        ctx.set_option(gatgpu.OPT_FUSE_NEXT_PROJECTION, 1)
        for l in range(3):
            ctx.set_norm(l, None, None)
