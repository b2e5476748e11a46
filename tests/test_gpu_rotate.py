"""Norms and rotation of queries and keys on the GPU against the plain computation in 64 bits."""
import math

import pytest
import torch

import gatgpu
from cache_cases import EPS, TYPE, generator, normal, rotate

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
HALVES, NEIGHBOURS = gatgpu.PAIRS_HALVES, gatgpu.PAIRS_NEIGHBOURS


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


class Problem:
    def __init__(self, rows, heads, kv_heads, dim, precision, rot=None, pairs=HALVES, norm=True, gammas=True, far=5000, seed=0, gap=0):
        g = generator(seed)
        self.shape = rows, heads, kv_heads, dim
        self.precision, self.rot, self.pairs, self.norm, self.eps = precision, dim if rot is None else rot, pairs, norm, 1e-5
        t = TYPE[precision]
        per = 8 if precision == BF else 4
        width = (heads + 2 * kv_heads) * dim + gap * per
        self.x = (normal(g, rows, width) * 2).to(t)  # queries, keys, values and a gap side by side
        self.dy = normal(g, rows, width).to(t)
        self.gamma = [1 + 0.3 * normal(g, dim) if gammas else None for _ in range(2)]
        self.position = torch.randint(0, far, (rows,), generator=g, dtype=torch.int32)
        self.freq = torch.pow(10000.0, -2.0 * torch.arange(max(1, self.rot // 2), dtype=torch.float64) / max(1, self.rot))[:self.rot // 2]

    def part(self, rows, which):
        n, h, hk, d = self.shape
        a = rows[:, :h * d] if which == 0 else rows[:, h * d:(h + hk) * d]
        return a.reshape(n, h if which == 0 else hk, d)

    def io(self, d, back=False):
        n, h, hk, dim = self.shape
        size, ld = d["x"].element_size(), d["x"].stride(0)
        at = h * dim * size
        io = gatgpu.RotateIO(precision=self.precision, heads=h, kv_heads=hk, dim=dim, norm=int(self.norm), rot=self.rot, pairs=self.pairs, eps=self.eps,
                             rows=n, q=d["x"].data_ptr(), k=d["x"].data_ptr() + at, q_stride=ld, k_stride=ld,
                             position=d["position"].data_ptr(), freq=d["freq"].data_ptr() if self.rot else None,
                             q_out=d["y"].data_ptr(), k_out=d["y"].data_ptr() + at, q_out_stride=ld, k_out_stride=ld)
        for name, gamma in zip(("gamma_q", "gamma_k"), d["gamma"]):
            setattr(io, name, None if gamma is None else gamma.data_ptr())
        if back:
            io.dq_out, io.dk_out, io.dq_out_stride, io.dk_out_stride = d["dy"].data_ptr(), d["dy"].data_ptr() + at, ld, ld
            io.dq, io.dk, io.dq_stride, io.dk_stride = d["dx"].data_ptr(), d["dx"].data_ptr() + at, ld, ld
            if self.norm:
                io.dgamma_q, io.dgamma_k = d["dgamma"][0].data_ptr(), d["dgamma"][1].data_ptr()
        return io

    def device(self, in_place=False):
        d = {"x": self.x.cuda(), "dy": self.dy.cuda(), "position": self.position.cuda(), "freq": self.freq.cuda(),
             "gamma": [None if g is None else g.cuda() for g in self.gamma]}
        d["y"] = d["x"] if in_place else torch.full_like(d["x"], 7.0)
        d["dx"] = d["dy"] if in_place else torch.full_like(d["x"], 7.0)
        d["dgamma"] = [torch.full((self.shape[3],), 7.0, device="cuda") for _ in range(2)]
        return d

    def run(self, ctx, back=True, in_place=False):
        d = self.device()
        if in_place:
            d["y"] = d["x"].clone()
            d["dx"] = d["dy"].clone()
            fwd, bwd = dict(d, x=d["y"]), dict(d, dy=d["dx"])
        else:
            fwd = bwd = d
        torch.cuda.synchronize()
        ctx.rotate_forward(self.io(fwd))
        if back:
            io = self.io(bwd, True)
            need = ctx.rotate_workspace(io)
            work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            ctx.rotate_backward(io, work.data_ptr(), need)
        ctx.synchronize()
        return d

    def check(self, got, back=True, in_place=False):
        n, h, hk, dim = self.shape
        ends = (h + hk) * dim
        if not in_place:  # values and the gap are nobody's
            assert bool((got["y"][:, ends:] == 7).all()) and (not back or bool((got["dx"][:, ends:] == 7).all()))
        step = 2.0 ** -24
        for which in range(2 if hk else 1):
            x = self.part(self.x, which).double().requires_grad_(True)
            gamma = self.gamma[which].double().requires_grad_(True) if self.gamma[which] is not None else None
            args = (self.eps, self.norm, self.position, self.freq, self.rot, self.pairs)
            y = rotate(x, gamma, *args)
            # Sums of magnitudes: |a| + |b| of each pair.
            def both(v):
                if not self.rot:
                    return v.abs()
                first = torch.arange(self.rot // 2) * (1 if self.pairs == HALVES else 2)
                second = first + (self.rot // 2 if self.pairs == HALVES else 1)
                m = v.abs().clone()
                m[..., first] = m[..., second] = v.abs()[..., first] + v.abs()[..., second]
                return m
            xd = x.detach()
            r = 1 / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + self.eps) if self.norm else torch.ones_like(xd[..., :1])
            g1 = gamma.detach().abs() if gamma is not None and self.norm else 1.0
            # The norm's factor (a sum of dim squares, a root, a quotient), three products, an angle rounded to 2^-25 of a turn, sine and cosine.
            rel = (dim / 2 + 12) * step + 2.0 ** -21
            tol = both(xd * r * g1) * rel + y.detach().abs() * EPS[self.precision] + 1e-37
            out = self.part(got["y"].cpu(), which).double()
            err = (out - y.detach()).abs()
            assert bool((err <= tol).all()), (which, float((err / tol).max()))
            if not back:
                continue
            dy = self.part(self.dy, which).double()
            wanted = [x] + ([gamma] if gamma is not None and self.norm else [])
            grads = torch.autograd.grad(y, wanted, dy)
            m = both(dy)
            nn = (xd * r).abs() if self.norm else torch.zeros_like(xd)
            g = m * g1
            rel = (2 * dim + 30) * step + 2.0 ** -20
            tol = r * (g + nn * (g * nn).mean(-1, keepdim=True)) * rel + grads[0].abs() * EPS[self.precision] + 1e-37
            err = (self.part(got["dx"].cpu(), which).double() - grads[0]).abs()
            assert bool((err <= tol).all()), (which, float((err / tol).max()))
            if self.norm:
                count = n * (h, hk)[which]
                want = grads[1] if gamma is not None else None
                if want is None:
                    unit = torch.ones(dim, dtype=torch.float64, requires_grad=True)
                    want = torch.autograd.grad(rotate(xd, unit, *args), unit, dy)[0]
                tol = (m * nn).sum((0, 1)) * ((count + dim + 40) * step + 2.0 ** -20) + 1e-37
                err = (got["dgamma"][which].cpu().double() - want).abs()
                assert bool((err <= tol).all()), (which, float((err / tol).max()))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("pairs", [HALVES, NEIGHBOURS])
@pytest.mark.parametrize("dim,rot", [(8, 8), (16, 4), (32, 32), (40, 40), (48, 24), (64, 64), (64, 20), (96, 48), (128, 128), (128, 2), (200, 200), (256, 256), (256, 0)])
def test_widths(ctx, precision, pairs, dim, rot):
    p = Problem(37, 6, 2, dim, precision, rot=rot, pairs=pairs, seed=dim + rot, gap=1)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("rows", [1, 2, 17, 300, 5000])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 4), (3, 0), (1, 7)])
def test_rows_and_heads(ctx, precision, rows, heads, kv_heads):
    p = Problem(rows, heads, kv_heads, 32, precision, seed=rows)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("norm,gammas", [(True, False), (False, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_without_gamma_or_norm_and_in_place(ctx, precision, norm, gammas, in_place):
    p = Problem(70, 5, 3, 64, precision, norm=norm, gammas=gammas, seed=4)
    p.check(p.run(ctx, in_place=in_place), in_place=in_place)
    p = Problem(70, 4, 2, 48, precision, rot=20, seed=5)  # pairs that are no whole chunks apart
    p.check(p.run(ctx, in_place=in_place), in_place=in_place)


@pytest.mark.parametrize("pairs", [HALVES, NEIGHBOURS])
def test_far_positions(ctx, pairs):
    """Angles of positions up to 2^31 keep their digits."""
    p = Problem(200, 2, 2, 64, FP, pairs=pairs, far=2 ** 31 - 1, seed=6)
    p.check(p.run(ctx))


def test_gradient_against_differences(ctx):
    """Of the plain form in 64 bits, in directions; h^2 / 6 of a third derivative of some hundreds is below 1e-7 of the slope."""
    p = Problem(9, 3, 2, 32, FP, rot=16, seed=8)
    got = p.run(ctx)
    g = generator(9)
    for which, h in ((0, 3), (1, 2)):
        x, gamma, dy = p.part(p.x, which).double(), p.gamma[which].double(), p.part(p.dy, which).double()
        args = (p.eps, True, p.position, p.freq, p.rot, p.pairs)
        dx, dgamma = p.part(got["dx"].cpu(), which).double(), got["dgamma"][which].cpu().double()
        for _ in range(4):
            u, w, step = normal(g, 9, h, 32).double(), normal(g, 32).double(), 1e-5
            slope = ((rotate(x + step * u, gamma + step * w, *args) - rotate(x - step * u, gamma - step * w, *args)) * dy).sum() / (2 * step)
            want = (dx * u).sum() + (dgamma * w).sum()
            size = (dx * u).abs().sum() + (dgamma * w).abs().sum()
            assert abs(float(slope - want)) < float(size) * 2.0 ** -19  # (32 columns: (2 dim + 30) 2^-24 + 2^-20)


def test_nan_and_infinity_stay_in_their_vector(ctx):
    p = Problem(20, 3, 2, 64, FP, seed=10)
    p.x[4, 64 + 3] = math.nan       # query head 1 of row 4
    p.x[5, 3 * 64 + 1] = math.inf   # key head 0 of row 5
    got = p.run(ctx, back=False)["y"].cpu()
    clean = Problem(20, 3, 2, 64, FP, seed=10)
    want = clean.run(ctx, back=False)["y"].cpu()
    same = torch.ones_like(got, dtype=torch.bool)
    same[4, 64:128] = False
    same[5, 192:256] = False
    assert torch.equal(got[same], want[same]) and bool(torch.isnan(got[4, 64:128]).all()) and not bool(torch.isfinite(got[5, 192:256]).all())


def test_equal_inputs_give_equal_bits_and_workspace_contents_do_not_matter(ctx):
    p = Problem(3000, 8, 2, 64, BF, seed=11)
    a, b = p.run(ctx), p.run(ctx)
    for n in ("y", "dx"):
        assert torch.equal(a[n], b[n])
    assert all(torch.equal(x, y) for x, y in zip(a["dgamma"], b["dgamma"]))


def test_captured_and_replayed(ctx):
    """Forward and backward in one graph, replayed on new inputs between eager calls."""
    p = Problem(50, 4, 2, 64, BF, seed=12)
    d = p.device()
    io = p.io(d, True)
    work = torch.empty(ctx.rotate_workspace(io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(ctx.stream())
    with torch.cuda.graph(graph, stream=stream):
        ctx.rotate_forward(io)
        ctx.rotate_backward(io, work.data_ptr(), work.numel())
    for seed in (13, 14, 15):
        q = Problem(50, 4, 2, 64, BF, seed=seed)
        q.gamma = p.gamma
        d["x"].copy_(q.x)
        d["dy"].copy_(q.dy)
        d["position"].copy_(q.position)
        for t in (d["y"], d["dx"], *d["dgamma"]):
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        q.check(d)
        p.check(p.run(ctx))


def test_no_rows_give_zeros(ctx):
    """Gradients of the norms' weights of no rows; arrays of no rows, and what only they would need, may be null."""
    p = Problem(1, 4, 2, 64, BF, seed=17)
    d = p.device()
    io = p.io(d, True)
    io.rows = 0
    for n in ("q", "k", "dq_out", "dk_out", "dq", "dk", "position", "freq"):
        setattr(io, n, None)
    work = torch.full((ctx.rotate_workspace(io),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.rotate_forward(io)
    ctx.rotate_backward(io, work.data_ptr(), work.numel())
    ctx.synchronize()
    assert all(bool((g == 0).all()) for g in d["dgamma"])


def test_refusals(ctx):
    p = Problem(10, 4, 2, 64, BF, seed=16)
    d = p.device()

    def refused(code=gatgpu.EINVAL, back=False, work=True, **change):
        io = p.io(d, True)
        for k, v in change.items():
            setattr(io, k, v)
        need = 1 << 20
        buffer = torch.empty(need, dtype=torch.uint8, device="cuda")
        with pytest.raises(gatgpu.GatGpuError) as err:
            if back:
                ctx.rotate_backward(io, buffer.data_ptr() if work is True else work, need if work is True else 16)
            else:
                ctx.rotate_forward(io)
        assert err.value.code == code, str(err.value)

    for change in (dict(precision=2), dict(heads=0), dict(heads=1025), dict(kv_heads=-1), dict(dim=12), dict(dim=264), dict(dim=0), dict(rot=3), dict(rot=66),
                   dict(rot=-2), dict(pairs=2), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(q=None), dict(k=None), dict(q_out=None),
                   dict(k_out=None), dict(position=None), dict(freq=None), dict(q_stride=255), dict(k_stride=127), dict(q_stride=2 ** 45),
                   dict(q=d["x"].data_ptr() + 2), dict(q_stride=d["x"].stride(0) + 1), dict(gamma_q=d["gamma"][0].data_ptr() + 2),
                   dict(freq=d["freq"].data_ptr() + 4), dict(position=d["position"].data_ptr() + 1), dict(q=p.x.data_ptr() // 16 * 16)):
        refused(**change)
    refused(code=gatgpu.EOVERFLOW, rows=2 ** 31)
    for change in (dict(dq_out=None), dict(dk=None), dict(q=None), dict(norm=0), dict(dgamma_q=d["dgamma"][0].data_ptr() + 1)):
        refused(back=True, **change)
    refused(back=True, work=None)
    refused(back=True, work=torch.empty(64, dtype=torch.uint8, device="cuda").data_ptr())  # too small
    with pytest.raises(gatgpu.GatGpuError):
        ctx.rotate_workspace(gatgpu.RotateIO(heads=1, dim=7))
    ctx.rotate_forward(gatgpu.RotateIO(heads=4, kv_heads=2, dim=64))  # no rows: nothing to read
