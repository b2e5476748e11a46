"""Layer norm on the GPU against the plain computation in 64 bits, alone and in the model's layers.

Bounds: u is the unit roundoff of FP32 (2^-24), t that of storage (2^-8 for bf16).  A row's mean
and centred square sum over W columns run in at most c = 2 ceil(W / threads) + 16 rounded
additions a term; the centred value is then off by (c + 2) u (|h| + mean |h|), n by that times
rstd plus (c + 8) u |n|, and so on through the formulas.
"""
import math

import numpy as np
import pytest
import torch

import gatgpu
import oracle
from gatgpu import inputs

pytestmark = pytest.mark.gpu

U, UB = 2.0 ** -24, 2.0 ** -8
WIDTHS = [1, 2, 7, 8, 100, 128, 129, 256, 257, 1000, 1024, 2047, 2048, 4096, 5001, 8192, 12000, 16384, 20001, 40000]


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


class Norm:
    def __init__(self, rows, width, precision, residual=True, elu=False, weights=True, pad=0, seed=0, eps=1e-5, mean=0.5):
        self.rows, self.width, self.precision, self.elu, self.eps = rows, width, precision, elu, eps
        self.t = torch.bfloat16 if precision == gatgpu.BF16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rand():
            x = torch.randn(max(rows, 1), width + pad, generator=g, device="cuda")
            return x.to(self.t)[:, :width]

        self.x = (rand().float() * 1.5 + mean).to(self.t) if not pad else rand()
        self.residual = rand() if residual else None
        self.dy, self.dsum = rand(), rand() if residual else None
        self.gamma = 1 + 0.3 * torch.randn(width, generator=g, device="cuda") if weights else None
        self.beta = 0.3 * torch.randn(width, generator=g, device="cuda") if weights else None

    def arrays(self):
        r, w = max(self.rows, 1), self.width
        out = {n: torch.full((r, w), 7.0, dtype=self.t, device="cuda") for n in ("y", "sum", "dx")}
        out.update({n: torch.full((r,), 7.0, device="cuda") for n in ("mean", "rstd")})
        out.update({n: torch.full((w,), 7.0, device="cuda") for n in ("dgamma", "dbeta")})
        io = gatgpu.NormIO(precision=self.precision, elu=int(self.elu), rows=self.rows, width=w, eps=self.eps,
                           x=self.x.data_ptr(), x_stride=self.x.stride(0), y=out["y"].data_ptr(), y_stride=w,
                           mean=out["mean"].data_ptr(), rstd=out["rstd"].data_ptr(), dy=self.dy.data_ptr(),
                           dy_stride=self.dy.stride(0), dx=out["dx"].data_ptr(), dx_stride=w,
                           dgamma=out["dgamma"].data_ptr(), dbeta=out["dbeta"].data_ptr())
        if self.gamma is not None:
            io.gamma, io.beta = self.gamma.data_ptr(), self.beta.data_ptr()
        if self.residual is not None:
            io.residual, io.residual_stride = self.residual.data_ptr(), self.residual.stride(0)
            io.sum, io.sum_stride = out["sum"].data_ptr(), w
            io.dsum, io.dsum_stride = self.dsum.data_ptr(), self.dsum.stride(0)
        else:
            del out["sum"]
        return out, io

    def run(self, ctx):
        out, io = self.arrays()
        ws = torch.empty(ctx.norm_workspace(self.rows, self.width), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        ctx.norm_forward(io)
        ctx.norm_backward(io, ws.data_ptr(), ws.numel())
        ctx.synchronize()
        return out

    def reference(self):
        h = self.x.double()
        val, tol = {}, {}
        t = UB if self.precision == gatgpu.BF16 else U
        if self.residual is not None:
            # (FP32 sums of two stored values, rounded to storage)
            h = (self.x.float() + self.residual.float()).to(self.t).double()
            val["sum"], tol["sum"] = h, torch.zeros_like(h)
        w = self.width
        c = 2 * math.ceil(w / 16) + 16 if w <= 4096 else 2 * math.ceil(w / 256) + 24
        gamma = torch.ones(w, dtype=torch.float64, device="cuda") if self.gamma is None else self.gamma.double()
        beta = torch.zeros(w, dtype=torch.float64, device="cuda") if self.beta is None else self.beta.double()
        mean = h.mean(1, keepdim=True)
        var = (h - mean).square().mean(1, keepdim=True)
        rstd = 1 / torch.sqrt(var + self.eps)
        n = (h - mean) * rstd
        off_mean = (c + 2) * U * h.abs().mean(1, keepdim=True)
        off_h = off_mean + 2 * U * (h - mean).abs()
        # relative error of var + eps: centred errors (twice), the sum's, and the square of the mean's own shift
        rel = ((2 * ((h - mean).abs() * off_h).mean(1, keepdim=True) + off_mean ** 2) / (var + self.eps)) + (c + 4) * U
        off_n = off_h * rstd + n.abs() * (rel + 4 * U)
        pre = n * gamma + beta
        off_pre = off_n * gamma.abs() + 3 * U * (pre.abs() + (n * gamma).abs())
        y = torch.where(pre >= 0, pre, torch.expm1(pre)) if self.elu else pre
        val.update(y=y, mean=mean.squeeze(1), rstd=rstd.squeeze(1))
        # ELU on the hardware exponential: 2e-6 of a value for bf16 rows, 4 u for FP32
        tol.update(y=off_pre + t * y.abs() + (3e-6 if t == UB else 8 * U) * y.abs(), mean=off_mean.squeeze(1),
                   rstd=(rstd * (rel + 4 * U)).squeeze(1))
        dt = self.dy.double()
        off_dt = torch.zeros_like(dt)
        if self.elu:
            slope = torch.where(pre < 0, torch.exp(pre), torch.ones_like(pre))
            off_dt = dt.abs() * torch.where(pre < off_pre, slope * (off_pre + 8 * U * (1 + pre.abs())) + 0, torch.zeros_like(pre))
            dt = dt * slope
        r = max(self.rows, 1)
        sums = (2 * math.ceil(r / 8) + 64) * U
        val["dgamma"], val["dbeta"] = (dt * n).sum(0), dt.sum(0)
        tol["dgamma"] = (off_dt * n.abs() + dt.abs() * off_n).sum(0) + sums * (dt * n).abs().sum(0)
        tol["dbeta"] = off_dt.sum(0) + sums * dt.abs().sum(0)
        g = dt * gamma
        off_g = off_dt * gamma.abs() + U * g.abs()
        s1, s2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
        off_1 = off_g.mean(1, keepdim=True) + (c + 2) * U * g.abs().mean(1, keepdim=True)
        off_2 = (off_g * n.abs() + g.abs() * off_n).mean(1, keepdim=True) + (c + 3) * U * (g * n).abs().mean(1, keepdim=True)
        inner = g - s1 - n * s2
        off_inner = off_g + off_1 + off_n * s2.abs() + n.abs() * off_2 + 4 * U * (g.abs() + s1.abs() + (n * s2).abs())
        dx = rstd * inner
        off = rstd * off_inner + (rel + 6 * U) * rstd * (g.abs() + s1.abs() + (n * s2).abs())
        if self.residual is not None:
            dx = dx + self.dsum.double()
            off = off + 2 * U * self.dsum.double().abs()
        val["dx"], tol["dx"] = dx, off + t * dx.abs()
        return val, tol

    def check(self, got):
        val, tol = self.reference()
        for name, want in val.items():
            if not self.rows:
                continue
            far = (got[name].double() - want).abs() - tol[name]
            assert bool(torch.isfinite(got[name]).all()), name
            assert float(far.max()) <= 1e-30, (name, float(far.max()))


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(ctx, precision, width):
    p = Norm(37, width, precision, residual=width % 2 == 0, elu=width % 3 == 0, seed=width)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("rows", [1, 3, 5, 1000, 20011])
@pytest.mark.parametrize("residual,elu,weights", [(False, False, True), (True, True, True), (True, False, False)])
def test_rows(ctx, precision, rows, residual, elu, weights):
    p = Norm(rows, 96, precision, residual, elu, weights, seed=rows)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("pad", [1, 8])
@pytest.mark.parametrize("width", [64, 257, 30001])
def test_strided_rows(ctx, precision, pad, width):
    p = Norm(9, width, precision, residual=True, elu=True, pad=pad, seed=pad)
    p.check(p.run(ctx))


def test_rows_around_a_large_mean(ctx):
    """The variance is that of the centred rows: a mean 1000 times the spread leaves it its digits."""
    p = Norm(64, 512, gatgpu.FP32, residual=False, mean=1500.0, seed=1)
    p.check(p.run(ctx))


def test_constant_rows(ctx):
    p = Norm(8, 256, gatgpu.FP32, residual=False, seed=2)
    p.x.fill_(3.0)
    got = p.run(ctx)
    assert torch.equal(got["y"], p.beta.expand(8, 256)) and torch.allclose(got["rstd"], torch.full((8,), 1e5 ** 0.5, device="cuda"))


@pytest.mark.parametrize("width", [256, 20001])
def test_bad_rows_stay_alone(ctx, width):
    p = Norm(40, width, gatgpu.BF16, residual=False, seed=3)
    want = p.run(ctx)
    p.x[7, 3], p.x[9, 0] = math.nan, math.inf
    got = p.run(ctx)
    keep = [r for r in range(40) if r not in (7, 9)]
    assert torch.equal(got["y"][keep], want["y"][keep]) and torch.equal(got["dx"][keep], want["dx"][keep])
    assert bool(torch.isnan(got["y"][7]).all())


@pytest.mark.parametrize("width", [256, 100, 40000])
def test_in_place(ctx, width):
    p = Norm(33, width, gatgpu.BF16, residual=True, elu=True, seed=4)
    want = p.run(ctx)
    x, res, dsum, dy = p.x.clone(), p.residual.clone(), p.dsum.clone(), p.dy.clone()
    out, io = p.arrays()
    io.x, io.residual, io.sum, io.y = x.data_ptr(), res.data_ptr(), res.data_ptr(), x.data_ptr()
    io.dsum, io.dx, io.dy = dsum.data_ptr(), dy.data_ptr(), dy.data_ptr()
    ws = torch.empty(ctx.norm_workspace(33, width), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.norm_forward(io)
    ctx.norm_backward(io, ws.data_ptr(), ws.numel())
    ctx.synchronize()
    assert torch.equal(x, want["y"]) and torch.equal(res, want["sum"]) and torch.equal(dy, want["dx"])
    assert torch.equal(out["dgamma"], want["dgamma"]) and torch.equal(out["dbeta"], want["dbeta"])


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("width", [3, 9, 131, 4099, 16001])
def test_in_place_at_widths_of_no_whole_loads(ctx, precision, width):
    """The row's last load begins before its place: its first columns are another thread's to write."""
    p = Norm(37, width, precision, residual=True, elu=True, seed=9)
    p.x[5, -2], p.dy[7, 0] = math.nan, math.inf
    want = p.run(ctx)
    bad = torch.zeros(37, dtype=torch.bool, device="cuda")
    bad[5] = True
    assert bool((torch.isfinite(want["y"]).all(1) == ~bad).all())
    bad[7] = True
    assert bool((torch.isfinite(want["dx"]).all(1) == ~bad).all())
    x, res, dsum, dy = p.x.clone(), p.residual.clone(), p.dsum.clone(), p.dy.clone()
    out, io = p.arrays()
    io.x, io.residual, io.sum, io.y = x.data_ptr(), res.data_ptr(), x.data_ptr(), res.data_ptr()
    io.dsum, io.dx, io.dy = dsum.data_ptr(), dsum.data_ptr(), dy.data_ptr()
    ws = torch.empty(ctx.norm_workspace(37, width), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.norm_forward(io)
    ctx.norm_backward(io, ws.data_ptr(), ws.numel())
    ctx.synchronize()
    for have, name in ((res, "y"), (x, "sum"), (dsum, "dx"), (out["dgamma"], "dgamma"), (out["dbeta"], "dbeta")):
        assert torch.equal(torch.nan_to_num(have, 5.0), torch.nan_to_num(want[name], 5.0)), name


def test_optional_arrays(ctx):
    p = Norm(50, 256, gatgpu.FP32, residual=True, seed=5)
    want = p.run(ctx)
    out, io = p.arrays()
    io.sum = io.mean = io.rstd = None
    torch.cuda.synchronize()
    ctx.norm_forward(io)
    ctx.synchronize()
    assert torch.equal(out["y"], want["y"]) and bool((out["sum"] == 7.0).all()) and bool((out["mean"] == 7.0).all())
    _, io = p.arrays()
    io.sum, io.mean, io.rstd = want["sum"].data_ptr(), want["mean"].data_ptr(), want["rstd"].data_ptr()
    io.dgamma = io.dbeta = None
    io.dx = out["dx"].data_ptr()
    ctx.norm_backward(io)
    ctx.synchronize()
    assert torch.equal(out["dx"], want["dx"])


def test_no_rows(ctx):
    p = Norm(0, 64, gatgpu.FP32, residual=False)
    got = p.run(ctx)
    assert bool((got["y"] == 7.0).all()) and bool((got["dgamma"] == 0).all()) and bool((got["dbeta"] == 0).all())


@pytest.mark.parametrize("width,rows", [(2, (1 << 28) + 5), (1040, (1 << 20) + 3), (4097, (1 << 20) + 3)])
def test_more_rows_than_one_grid_dimension_takes(ctx, width, rows):
    """In place; more than 2^32 threads, and more than 2^20 blocks of a row each."""
    x = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda").fill_(3.0)
    at = torch.tensor([0, 1, (1 << 20) - 1, rows // 2, rows - 2, rows - 1], device="cuda")
    x[at] = torch.randn(at.numel(), width, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").to(torch.bfloat16)
    h = x[at].double()
    io = gatgpu.NormIO(precision=gatgpu.BF16, rows=rows, width=width, eps=1e-5, x=x.data_ptr(), x_stride=width,
                       y=x.data_ptr(), y_stride=width)
    torch.cuda.synchronize()
    ctx.norm_forward(io)
    ctx.synchronize()
    want = (h - h.mean(1, keepdim=True)) / torch.sqrt(h.var(1, unbiased=False, keepdim=True) + 1e-5)
    # FP32 sums of at most 4097 columns by 16 threads or more, values of at most 6, beside the stored rounding
    assert float(((x[at].double() - want).abs() - UB * want.abs()).max()) <= 600 * U * 36
    # (a constant row's norm is 0 up to its mean's rounding, 3 u, over sqrt(eps))
    assert sum(int((part.abs() > 1e-2).any(1).sum()) for part in x.split(1 << 24)) == at.numel()


def test_gradients_against_differences(ctx):
    p = Norm(20, 48, gatgpu.FP32, residual=False, elu=True, seed=6)
    got = p.run(ctx)
    g = torch.Generator(device="cuda").manual_seed(7)

    def loss(x, gamma, beta):
        y = torch.nn.functional.layer_norm(x, (48,), gamma, beta, p.eps)
        return float((torch.nn.functional.elu(y) * p.dy.double()).sum())

    at = [p.x.double(), p.gamma.double(), p.beta.double()]
    for k, name in enumerate(("dx", "dgamma", "dbeta")):
        d = torch.randn(at[k].shape, generator=g, device="cuda", dtype=torch.float64)
        moved = [[x + s * 1e-5 * d if i == k else x for i, x in enumerate(at)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / 2e-5
        # (ELU's second derivative jumps at 0: a crossing changes a difference by at most step |d|^2 |dy|)
        assert abs(slope - float((got[name].double() * d).sum())) < 1e-4 * (1 + abs(slope)), name


def test_same_bits_and_replay(ctx):
    p = Norm(5003, 320, gatgpu.BF16, residual=True, elu=True, seed=8)
    a, b = p.run(ctx), p.run(ctx)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    stream = torch.cuda.ExternalStream(ctx.stream())
    out, io = p.arrays()
    ws = torch.empty(ctx.norm_workspace(p.rows, p.width), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        ctx.norm_forward(io)
        ctx.norm_backward(io, ws.data_ptr(), ws.numel())
    for k in range(3):
        p.x.copy_(torch.randn(p.x.shape, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = p.run(ctx)
        for n in want:
            assert torch.equal(out[n], want[n]), (k, n)


def test_refusals(ctx):
    p = Norm(8, 64, gatgpu.BF16, residual=True, seed=9)
    host = torch.empty(4096)
    ws = torch.empty(ctx.norm_workspace(8, 64), dtype=torch.uint8, device="cuda")

    def refused(call, code=gatgpu.EINVAL, **change):
        _, io = p.arrays()
        for n, x in change.items():
            setattr(io, n, x)
        with pytest.raises(gatgpu.GatGpuError) as err:
            call(io)
        assert err.value.code == code, change

    back = lambda io: ctx.norm_backward(io, ws.data_ptr(), ws.numel())  # noqa: E731
    for call in (ctx.norm_forward, back):
        refused(call, precision=2)
        refused(call, width=0)
        refused(call, eps=-1.0)
        refused(call, eps=math.nan)
        refused(call, rows=1 << 31, code=gatgpu.EOVERFLOW)
        refused(call, gamma=host.data_ptr())
    for n in ("x", "y"):
        refused(ctx.norm_forward, **{n: None})
        refused(ctx.norm_forward, **{n: host.data_ptr()})
        refused(ctx.norm_forward, **{n: p.x.data_ptr() + 1})
        refused(ctx.norm_forward, **{n + "_stride": 63})
    refused(ctx.norm_forward, residual=None)  # sum without one
    for n in ("dy", "dx", "mean", "rstd", "sum"):
        refused(back, **{n: None})
    refused(lambda io: ctx.norm_backward(io, ws.data_ptr(), ws.numel() - 1))
    refused(lambda io: ctx.norm_backward(io, host.data_ptr() // 16 * 16 + 16, 1 << 20))
    with pytest.raises(gatgpu.GatGpuError):
        ctx.lib.gatgpu_norm_forward(ctx.h, None)
        ctx._check(ctx.lib.gatgpu_norm_forward(ctx.h, None))


# ---- the model's own layers
def model_norms(model, seed):
    rng = np.random.default_rng(seed)
    widths = [p["heads"] * p["dim"] for p in model]
    return [((1 + 0.3 * rng.standard_normal(w)).astype(np.float32), (0.3 * rng.standard_normal(w)).astype(np.float32)) for w in widths]


def plain_norm(x, gamma, beta, eps, hidden):
    x = x.astype(np.float64)
    c = x - x.mean(1, keepdims=True)
    y = c / np.sqrt((c * c).mean(1, keepdims=True) + eps) * gamma + beta
    return np.where(y >= 0, y, np.expm1(y)) if hidden else y


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("dataflow", [gatgpu.TRANSFORM_FIRST, gatgpu.AGGREGATE_FIRST])
@pytest.mark.parametrize("fuse", [0, 2])
def test_norm_in_the_model(ctx, precision, dataflow, fuse):
    """Every layer: norm and ELU of what the layer gives without them, on the same input; the chained
    model gives what its layers give one after another; without norms it gives what it gave before."""
    if precision == gatgpu.FP32 and dataflow == gatgpu.AGGREGATE_FIRST:
        pytest.skip("aggregate-first layers are bf16")
    row, col = inputs.powerlaw_graph(3000, 40000, 600, 5)
    x = inputs.normal((3000, 100), 6)
    model = inputs.glorot_model(100, 8, 32, 47, 7)
    norms = model_norms(model, 8)
    ctx.set_graph(row, col)
    ctx.set_model(model)
    ctx.set_input(x)
    ctx.set_option(gatgpu.OPT_FUSE_NEXT_PROJECTION, fuse)
    try:
        before = ctx.model_forward(precision, dataflow)[0]
        h = x
        for l in range(3):
            flow = dataflow if l == 0 else gatgpu.TRANSFORM_FIRST
            ctx.layer_forward(l, precision, flow, False, input=h)
            raw = ctx.stage(l, "out")
            ctx.set_norm(l, *norms[l], 1e-5)
            ctx.layer_forward(l, precision, flow, l < 2, input=h)
            out = ctx.stage(l, "out")
            want = plain_norm(raw, *norms[l], 1e-5, l < 2)
            # FP32 over at most 256 columns: 300 u of a value of at most 16 times gamma
            assert np.abs(out - want).max() < 300 * U * 16 * 2.5
            h = out
        for l in range(3):
            ctx.set_norm(l, *norms[l], 1e-5)
        logits = ctx.model_forward(precision, dataflow)[0]
        if dataflow == gatgpu.TRANSFORM_FIRST:
            assert np.array_equal(logits, h)
        assert np.array_equal(ctx.stage(1, "out"), ctx.stage(1, "out")) and ctx.has_stage(1, "out")
        ctx.set_norm(1, None, None)  # layer 1's aggregation may carry layer 2's projection again
        one = ctx.model_forward(precision, dataflow)[0]
        assert not np.array_equal(one, logits) and np.isfinite(one).all()
        for l in (0, 2):
            ctx.set_norm(l, None, None)
        assert np.array_equal(ctx.model_forward(precision, dataflow)[0], before)
    finally:
        ctx.set_option(gatgpu.OPT_FUSE_NEXT_PROJECTION, 1)
        for l in range(3):
            ctx.set_norm(l, None, None)


@pytest.mark.parametrize("precision", [gatgpu.FP32, gatgpu.BF16])
@pytest.mark.parametrize("shift", [0, 4])
def test_norm_in_the_static_layer(ctx, precision, shift):
    row, col = inputs.powerlaw_graph(2000, 30000, 500, 9)
    x = inputs.normal((2000, 64), 10)
    p = inputs.glorot_param(64, 8, 32, 11)
    gamma, beta = model_norms([p], 12)[0]
    ctx.set_graph(row, col)
    ctx.set_layer(0, p)
    ctx.set_norm(0, gamma, beta)
    try:
        assert 0 < ctx.static_scratch_need(0, precision, True) == ctx.static_scratch_need(0, precision, False)
        ctx.layer_forward(0, precision, gatgpu.TRANSFORM_FIRST, True, input=x)
        want = ctx.stage(0, "out")
        xd = torch.from_numpy(x).cuda()
        od = torch.full((2000 * 256 + 4,), 7.0, device="cuda")
        torch.cuda.synchronize()
        ctx.layer_forward_static(0, precision, True, xd.data_ptr(), od.data_ptr() + shift)
        ctx.synchronize()
        assert np.array_equal(od[shift // 4:][:2000 * 256].view(2000, 256).cpu().numpy(), want)
    finally:
        ctx.set_norm(0, None, None)


def test_set_norm_refusals(ctx):
    row, col = inputs.uniform_graph(200, 4, 1)
    p = inputs.glorot_param(16, 2, 8, 2)
    good = np.ones(16, np.float32)
    with gatgpu.Context(0) as fresh:
        with pytest.raises(gatgpu.GatGpuError) as err:
            fresh.set_norm(0, good, good)
        assert err.value.code == gatgpu.ESTATE
        fresh.set_graph(row, col)
        fresh.set_layer(0, p)
        for args, code in [((3, good, good, 1e-5), gatgpu.EINVAL), ((0, good, good, -1.0), gatgpu.EINVAL),
                           ((0, good * np.nan, good, 1e-5), gatgpu.ENONFINITE), ((0, good, good * np.inf, 1e-5), gatgpu.ENONFINITE)]:
            if args[0] == 3:
                with pytest.raises(gatgpu.GatGpuError) as err:
                    fresh._check(fresh.lib.gatgpu_set_norm(fresh.h, 3, good.ctypes.data, good.ctypes.data, 1e-5))
            else:
                with pytest.raises(gatgpu.GatGpuError) as err:
                    fresh.set_norm(*args)
            assert err.value.code == code
        with pytest.raises(gatgpu.GatGpuError):
            fresh._check(fresh.lib.gatgpu_set_norm(fresh.h, 0, good.ctypes.data, None, 1e-5))
        with pytest.raises(ValueError):
            fresh.set_norm(0, good[:8], good[:8])
        fresh.set_norm(0, good, good)
        x = inputs.normal((200, 16), 3)
        fresh.layer_forward(0, gatgpu.FP32, hidden=False, input=x)
        normed = fresh.stage(0, "out")
        fresh.set_layer(0, p)  # new weights: no norm
        fresh.layer_forward(0, gatgpu.FP32, hidden=False, input=x)
        assert not np.array_equal(fresh.stage(0, "out"), normed)
