"""Segment attention on the GPU against the plain computation in 64 bits (attention_cases.py)."""
import math

import numpy as np
import pytest
import torch

import gatgpu
from attention_cases import HIDDEN, Problem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
FULL, PREFIX = gatgpu.MASK_FULL, gatgpu.MASK_PREFIX
NONE, LINEAR, TABLE = gatgpu.BIAS_NONE, gatgpu.BIAS_LINEAR, gatgpu.BIAS_TABLE
ODD = [1, 31, 32, 33, 0, 64, 65, 100, 2]


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128])
def test_self_attention_lengths(ctx, precision, dim):
    p = Problem(ODD, ODD, 2, 2, dim, precision, seed=dim, gap=3)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 2), (8, 1), (5, 1)])
@pytest.mark.parametrize("bias,buckets", [(NONE, 0), (LINEAR, 0), (TABLE, 7)])
def test_shared_heads(ctx, precision, heads, kv_heads, bias, buckets):
    p = Problem([40, 7, 1], [40, 90, 33], heads, kv_heads, 32, precision, mask=PREFIX, prefix=[5, 0, 20], bias=bias,
                buckets=buckets, seed=heads)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("mask", [FULL, PREFIX])
@pytest.mark.parametrize("bias,buckets", [(NONE, 0), (LINEAR, 0), (TABLE, 1), (TABLE, 64)])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_masks_biases_caps(ctx, precision, mask, bias, buckets, cap):
    p = Problem([70, 129, 16], [70, 129, 50], 4, 2, 64, precision, mask=mask, prefix=[33, 0, 50], bias=bias,
                buckets=buckets, cap=cap, seed=3)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_many_rows_share_tiles(ctx, precision, dim):
    """Enough rows for blocks of four waves, in both passes."""
    lens = [200, 513, 128, 1, 96] + [384] * 12
    p = Problem(lens, lens, 32, 16, dim, precision, mask=PREFIX, prefix=[0, 300, 128, 0, 40] + [0] * 12, bias=LINEAR, cap=5.0, seed=1)
    p.check(p.run(ctx))


def test_many_rows_with_a_table(ctx):
    lens = [200, 513, 128, 1, 96] + [384] * 12
    p = Problem(lens, lens, 32, 32, 32, BF, bias=TABLE, buckets=20, seed=2)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("heads,kv_heads,q_len", [(8, 8, 1), (32, 4, 1), (8, 1, 3), (8, 2, 9)])
@pytest.mark.parametrize("bias,buckets", [(LINEAR, 0), (TABLE, 9)])
def test_new_tokens_over_long_keys(ctx, precision, heads, kv_heads, q_len, bias, buckets):
    """Few rows over many keys: ranges of keys, joined."""
    p = Problem([q_len] * 4, [1, 3000, 257, 5001], heads, kv_heads, 64, precision, mask=PREFIX, bias=bias, buckets=buckets, seed=5)
    assert p.plan(ctx).workspace_bytes() > 0
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_rows_that_see_nothing(ctx, precision):
    """More queries than keys under the causal mask, no keys at all, and hidden pairs."""
    p = Problem([50, 20, 40], [30, 0, 40], 2, 2, 32, precision, mask=PREFIX, seed=6)
    got = p.run(ctx)
    assert bool((got["out"][:20] == 0).all()) and bool((got["lse"][:20] == -math.inf).all())
    p.check(got)
    p = Problem([40, 33], [40, 70], 2, 1, 64, precision, bias=TABLE, buckets=5, seed=7)
    p.distances(0)[3] = HIDDEN
    p.distances(0)[:, 9] = HIDDEN
    p.distances(1)[:] = HIDDEN
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_table_of_minus_infinity_hides(ctx, precision):
    p = Problem([65], [65], 2, 2, 32, precision, bias=TABLE, buckets=6, seed=8)
    p.table[0, 2] = -math.inf
    p.table[1] = -math.inf
    got = p.run(ctx)
    assert bool((got["dbias"][1] == 0).all()) and float(got["dbias"][0, 2]) == 0
    p.check(got)


@pytest.mark.parametrize("lowest", [-3.0e38, -1.0e30, -1.0e9, -1.0e6])
def test_table_of_lowest_values(ctx, lowest):
    """A table entry of the type's lowest value, in place of a mask: row 7 has nothing else."""
    p = Problem([40], [40], 2, 2, 32, FP, bias=TABLE, buckets=4, hidden=0.0, seed=9)
    p.table[:, 1:] = lowest
    p.distances(0)[:] = 0
    p.distances(0)[:, 20:] = 2
    p.distances(0)[7] = 3
    got = p.run(ctx)
    assert bool((got["out"][7] == 0).all()) and bool((got["lse"][7] == -math.inf).all())
    p.check(got)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("many", [False, True])
def test_values_that_nobody_sees(ctx, precision, value, many):
    """NaN and infinities outside the segments and in nodes without an edge reach nothing."""
    lens = [70, 40] + ([384] * 22 if many else [])
    heads = 32 if many else 2
    clean = Problem(lens, lens, heads, heads, 32, precision, bias=TABLE, buckets=5, seed=10, gap=5)
    for s, n in ((0, 9), (0, 69), (1, 0)):
        clean.distances(s)[n] = HIDDEN
        clean.distances(s)[:, n] = HIDDEN
    want = clean.run(ctx)
    for s, n in ((0, 9), (0, 69), (1, 0)):
        for x, b in ((clean.q, clean.q_begin), (clean.k, clean.k_begin), (clean.v, clean.k_begin), (clean.dout, clean.q_begin)):
            x[int(b[s]) + n] = value
    for x in (clean.q, clean.k, clean.v, clean.dout):
        x[:5] = value
        x[75:80] = value
        x[-5:] = value
    got = clean.run(ctx)
    for name in want:
        assert torch.equal(want[name], got[name]), name


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_bad_value_reaches_the_rows_that_see_it(ctx, precision, value):
    """Causal mask, one element of a value row: rows before it are as they were, rows from it on hold it."""
    p = Problem([100], [100], 2, 2, 32, precision, mask=PREFIX, seed=11)
    want = p.run(ctx, train=False)["out"]
    p.v[60, 1, 5] = value
    got = p.run(ctx, train=False)["out"]
    assert torch.equal(got[:60], want[:60]) and torch.equal(got[:, 0], want[:, 0])
    column = got[60:, 1, 5].float()
    assert bool(torch.isnan(column).all()) if math.isnan(value) else bool((column == value).all())
    keep = [c for c in range(32) if c != 5]
    assert torch.equal(got[60:, 1, keep], want[60:, 1, keep])


def test_both_infinities_make_nan(ctx):
    p = Problem([40], [40], 1, 1, 32, BF, seed=12)
    p.v[3, 0, 0], p.v[30, 0, 0] = math.inf, -math.inf
    got = p.run(ctx, train=False)["out"]
    assert bool(torch.isnan(got[:, 0, 0]).all()) and bool(torch.isfinite(got[:, 0, 1:]).all())


@pytest.mark.parametrize("precision", [FP, BF])
def test_bad_gradients_stay_with_their_rows(ctx, precision):
    """A NaN in dout of one row: its own dq, and dk and dv of the keys that it sees, and no others."""
    p = Problem([90], [90], 2, 2, 32, precision, mask=PREFIX, seed=13)
    want = p.run(ctx)
    p.dout[50, 0, 3] = math.nan
    got = p.run(ctx)
    assert bool(torch.isnan(got["dq"][50, 0]).all())
    assert bool(torch.isnan(got["dk"][:51, 0]).all()) and bool(torch.isnan(got["dv"][:51, 0, 3]).all())
    other = [r for r in range(90) if r != 50]
    assert torch.equal(got["dq"][other], want["dq"][other])
    for n in ("dk", "dv"):
        assert torch.equal(got[n][51:], want[n][51:]) and torch.equal(got[n][:, 1], want[n][:, 1])


@pytest.mark.parametrize("bias,cap", [(NONE, 0.0), (TABLE, 2.0), (LINEAR, 4.0)])
def test_gradients_against_differences(ctx, bias, cap):
    """The plain function in 64 bits, moved both ways along random directions."""
    p = Problem([40, 9], [40, 30], 4, 2, 32, FP, mask=PREFIX, prefix=[10, 0], bias=bias, buckets=6 if bias == TABLE else 0, cap=cap, seed=14)
    got = p.run(ctx)
    _, tol = p.reference()

    def loss(x):
        total = 0.0
        for s in range(2):
            for h in range(4):
                a = p.segment(s, h, x)
                w, _ = p.weights(a)
                total += float((torch.matmul(w, a["v"]) * p.dout[a["qa"]:a["qa"] + a["nq"], h].double()).sum())
        return total

    g = torch.Generator(device="cuda").manual_seed(1)
    names = [("q", "dq"), ("k", "dk"), ("v", "dv")] + ([("table", "dbias")] if bias == TABLE else [])
    for name, grad in names:
        x = getattr(p, name).double()
        d = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
        step = 1e-5  # third derivatives of order 100 leave 1e-8; the loss's own rounding 1e-10
        slope = (loss({name: x + step * d}) - loss({name: x - step * d})) / (2 * step)
        mine = float((got[grad].double() * d).sum())
        assert abs(slope - mine) <= float((tol[grad] * d.abs()).sum()) + 1e-6 * abs(slope) + 1e-6, (name, slope, mine)


@pytest.mark.parametrize("precision", [FP, BF])
def test_same_bits_twice_and_without_training_arrays(ctx, precision):
    p = Problem([300, 77], [300, 200], 8, 4, 64, precision, bias=TABLE, buckets=12, cap=9.0, seed=15)
    a, b = p.run(ctx), p.run(ctx)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    with p.plan(ctx) as plan:
        out, io = p.buffers(train=False)
        rest = torch.empty_like(out["out"])  # (with it the weights keep 16 bits, so out may round otherwise without it)
        io.lse = None
        if precision == BF:
            io.rest = rest.data_ptr()
        ws = torch.empty(max(1, plan.workspace_bytes()), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        plan.forward(io, ws.data_ptr(), ws.numel())
        ctx.synchronize()
    assert torch.equal(out["out"], a["out"]) and bool((out["lse"] == 7.0).all())
    p.check(p.run(ctx, train=False), train=False)


def test_shared_key_rows(ctx):
    """Two segments over one prefix of a cache: forward as usual, no backward."""
    p = Problem([3, 2], [400, 400], 4, 2, 64, BF, seed=16)
    p.k_begin = np.array([0, 0])
    p.check(p.run(ctx, train=False), train=False)
    with pytest.raises(gatgpu.GatGpuError) as err:
        p.run(ctx)
    assert err.value.code == gatgpu.EINVAL and "overlap" in str(err.value)


def test_no_segments_and_no_rows(ctx):
    for lens in ([], [0, 0]):
        p = Problem(lens, lens, 2, 2, 32, BF, bias=TABLE, buckets=3, seed=17)
        got = p.run(ctx)
        assert bool((got["out"] == 7.0).all()) and bool((got["dbias"] == 0).all())
    p = Problem([0, 4], [40, 4], 2, 2, 32, BF, seed=18)  # keys without a query: their gradients are 0
    got = p.run(ctx)
    assert bool((got["dk"][:40] == 0).all()) and bool((got["dv"][:40] == 0).all())
    p.check(got)


def test_distance_layout(ctx):
    p = Problem([5, 0, 33], [17, 40, 33], 2, 2, 32, BF, bias=TABLE, buckets=3)
    with p.plan(ctx) as plan:
        size, off, ld = plan.distance_layout()
    assert size == p.off[-1] and list(off) == list(p.off[:-1]) and list(ld) == p.ld


def test_captured_calls_replay(ctx):
    """Forward and backward in one graph, replayed on new inputs, with eager calls between."""
    p = Problem([130, 40], [130, 700], 8, 2, 64, BF, mask=PREFIX, bias=TABLE, buckets=9, cap=6.0, seed=19)
    stream = torch.cuda.ExternalStream(ctx.stream())
    with p.plan(ctx) as plan:
        out, io = p.buffers()
        need = max(1, plan.workspace_bytes(), plan.workspace_bytes(backward=True))
        ws, other = (torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        plan.forward(io, ws.data_ptr(), need)
        plan.backward(io, ws.data_ptr(), need)
        ctx.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            plan.forward(io, ws.data_ptr(), need)
            plan.backward(io, ws.data_ptr(), need)
        g = torch.Generator(device="cuda").manual_seed(2)
        for _ in range(4):
            for x in (p.q, p.k, p.v, p.dout):
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            for x in out.values():
                x.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            eager, eio = p.buffers()
            torch.cuda.synchronize()
            plan.forward(eio, other.data_ptr(), need)
            plan.backward(eio, other.data_ptr(), need)
            ctx.synchronize()
            for n in out:
                assert torch.equal(out[n], eager[n]), n
    p.check(eager)


def test_two_calls_in_flight(ctx):
    """Two plans of two contexts at once, a workspace each."""
    problems = [Problem([1] * 8, [4000] * 8, 8, 8, 64, BF, seed=s) for s in (20, 21)]
    alone = [p.run(ctx, train=False)["out"] for p in problems]
    with gatgpu.Context(0) as second:
        plans = [problems[0].plan(ctx), problems[1].plan(second)]
        made = [p.buffers(train=False) for p in problems]
        ws = [torch.empty(plan.workspace_bytes(), dtype=torch.uint8, device="cuda") for plan in plans]
        torch.cuda.synchronize()
        for _ in range(5):
            for plan, (_, io), w in zip(plans, made, ws):
                plan.forward(io, w.data_ptr(), w.numel())
        torch.cuda.synchronize()
        for plan in plans:
            plan.close()
    for (out, _), want in zip(made, alone):
        assert torch.equal(out["out"], want)


def test_far_rows(ctx):
    """Keys behind 2^32 bytes of a cache."""
    p = Problem([2], [700], 4, 4, 64, BF, mask=PREFIX, seed=22)
    want = p.run(ctx, train=False)["out"]
    rows = (1 << 32) // (2 * 4 * 64 * 2) + 1000
    cache = torch.zeros(rows, 8, 64, dtype=torch.bfloat16, device="cuda")
    cache[-700:, :4], cache[-700:, 4:] = p.k, p.v
    p.k, p.v = cache[:, :4], cache[:, 4:]
    p.k_begin = np.array([rows - 700])
    assert torch.equal(p.run(ctx, train=False)["out"], want)


def test_refusals(ctx):
    def plan(**change):
        a = dict(q_len=[4, 4], k_len=[4, 4], heads=4, kv_heads=2, dim=32, precision=BF)
        a.update(change)
        return gatgpu.Attention(ctx, a.pop("q_len"), a.pop("k_len"), **a)

    for change, code in [
            (dict(heads=65, kv_heads=65), gatgpu.EINVAL), (dict(heads=4, kv_heads=3), gatgpu.EINVAL), (dict(heads=0, kv_heads=1), gatgpu.EINVAL),
            (dict(kv_heads=0), gatgpu.EINVAL), (dict(dim=12), gatgpu.EINVAL), (dict(dim=136), gatgpu.EINVAL), (dict(dim=0, scale=1.0), gatgpu.EINVAL),
            (dict(precision=2), gatgpu.EINVAL), (dict(mask=2), gatgpu.EINVAL), (dict(bias=3), gatgpu.EINVAL),
            (dict(bias=TABLE, buckets=0), gatgpu.EINVAL), (dict(bias=TABLE, buckets=65), gatgpu.EINVAL),
            (dict(scale=0.0), gatgpu.EINVAL), (dict(scale=-1.0), gatgpu.EINVAL), (dict(scale=math.nan), gatgpu.EINVAL),
            (dict(cap=-1.0), gatgpu.EINVAL), (dict(cap=math.inf), gatgpu.EINVAL), (dict(q_begin=[0, 3]), gatgpu.EINVAL),
            (dict(q_len=[1 << 30, 1], q_begin=[0, 1 << 31]), gatgpu.EOVERFLOW), (dict(k_len=[(1 << 30) + 1, 1]), gatgpu.EOVERFLOW),
            (dict(k_begin=[0, 1 << 50]), gatgpu.EOVERFLOW)]:
        with pytest.raises(gatgpu.GatGpuError) as err:
            plan(**change)
        assert err.value.code == code, change
    p = Problem([40], [300], 4, 2, 64, BF, bias=TABLE, buckets=5, seed=23)
    with p.plan(ctx) as made:
        need = max(1, made.workspace_bytes(), made.workspace_bytes(backward=True))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        host = torch.empty(1 << 16, dtype=torch.float32)
        out, _ = p.buffers()

        def refused(call, size=need, at=None, **change):
            _, io = p.buffers()
            for n, x in change.items():
                setattr(io, n, x)
            with pytest.raises(gatgpu.GatGpuError) as err:
                call(io, ws.data_ptr() if at is None else at, size)
            assert err.value.code == gatgpu.EINVAL, change

        base, width = p.q.data_ptr(), 4 * 64
        for call in (made.forward, made.backward):
            for n in ("q", "k", "v", "out", "bias", "dist"):
                refused(call, **{n: None})
                refused(call, **{n: base + 2})
                refused(call, **{n: host.data_ptr() // 16 * 16})
            for n in ("q_stride", "out_stride"):
                refused(call, **{n: width - 8})
                refused(call, **{n: width + 4})
            refused(call, k_stride=64)
        refused(made.backward, size=0)
        refused(made.backward, at=host.data_ptr() // 16 * 16 + 16)
        for n in ("dout", "dq", "dk", "dv", "lse"):
            refused(made.backward, **{n: None})
        refused(made.backward, rest=None)
        refused(made.backward, dbias=base + 2)
    q = Problem([1], [20000], 4, 2, 64, BF, seed=26)  # its keys are cut into ranges that need a workspace
    with q.plan(ctx) as made:
        _, io = q.buffers(train=False)
        need = made.workspace_bytes()
        assert need > 0
        for at, size in ((ws.data_ptr(), need - 1), (None, need), (host.data_ptr() // 16 * 16 + 16, need), (ws.data_ptr() + 8, need)):
            with pytest.raises(gatgpu.GatGpuError) as err:
                made.forward(io, at, size)
            assert err.value.code == gatgpu.EINVAL
    q = Problem([4], [4], 2, 2, 32, FP, seed=24)
    with q.plan(ctx) as made, pytest.raises(gatgpu.GatGpuError):
        _, io = q.buffers()
        io.rest = io.out
        made.forward(io)
    with pytest.raises(gatgpu.GatGpuError):
        made_lin = Problem([4], [4], 2, 2, 32, FP, bias=LINEAR, seed=25)
        with made_lin.plan(ctx) as made:
            made.distance_layout()


def test_the_current_device_stays(ctx):
    before = torch.cuda.current_device()
    p = Problem([4], [4], 2, 2, 32, FP, seed=26)
    p.run(ctx)
    assert torch.cuda.current_device() == before


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_len,bias,buckets", [(8, 8, 1, LINEAR, 0), (32, 2, 1, NONE, 0), (6, 2, 3, TABLE, 9), (40, 1, 2, TABLE, 64)])
def test_waves_cut_the_keys(ctx, precision, dim, heads, kv_heads, q_len, bias, buckets):
    """Few rows over some hundred keys: the waves of a block take a range each, some of them none."""
    keys = [300, 33, 1, 0, 380, 97]
    p = Problem([q_len] * 6, keys, heads, kv_heads, dim, precision, mask=PREFIX, bias=bias, buckets=buckets, cap=4.0, seed=31, gap=2)
    if heads < 40:  # (a table for 40 heads leaves the widest tiles no room: tasks, joined by a launch)
        assert p.plan(ctx).workspace_bytes() == 0
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_bad_values_where_waves_cut_the_keys(ctx, precision, value):
    """The first query sees no bad key, the second one of them."""
    p = Problem([2, 1], [290, 310], 4, 2, 64, precision, mask=PREFIX, seed=32)
    p.v[289, 1, 5] = value
    p.k[290 + 100, 0, 3] = math.nan
    p.check(p.run(ctx, train=False), train=False)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,bias,buckets,cap", [(3, 1, LINEAR, 0, 3.0), (8, 1, TABLE, 5, 0.0), (2, 2, TABLE, 64, 0.0), (4, 2, NONE, 0, 2.0)])
def test_segments_of_up_to_128_keys(ctx, precision, dim, heads, kv_heads, bias, buckets, cap):
    """Every number of waves of the short segments' backward pass, and lengths at its edges."""
    lens = [32, 33, 64, 65, 96, 97, 128, 129]
    p = Problem([32, 5, 70, 65, 1, 97, 40, 20], lens, heads, kv_heads, dim, precision, mask=PREFIX, prefix=[10] * 8, bias=bias,
                buckets=buckets, cap=cap, seed=33)
    p.check(p.run(ctx))


@pytest.mark.parametrize("dim", [32, 64])
@pytest.mark.parametrize("bias,buckets", [(TABLE, 6), (LINEAR, 0)])
def test_many_short_segments(ctx, dim, bias, buckets):
    """So many that a wave takes several heads of a segment, and two blocks of keys."""
    keys = [34 + i % 31 for i in range(56)] + [1 + i % 32 for i in range(140)]
    p = Problem([n if i % 3 else 2 for i, n in enumerate(keys)], keys, 64, 64, dim, BF, bias=bias, buckets=buckets, seed=34)
    p.check(p.run(ctx, train=False), train=False)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim", [24, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,bias,buckets,cap", [(8, 1, LINEAR, 0, 3.0), (3, 1, TABLE, 9, 0.0), (2, 2, NONE, 0, 0.0)])
def test_few_long_segments(ctx, precision, dim, heads, kv_heads, bias, buckets, cap):
    """Few blocks: the backward passes take ranges of a tile's keys and of its rows, which are joined."""
    p = Problem([700, 1, 1100], [1090, 900, 1100], heads, kv_heads, dim, precision, mask=PREFIX, prefix=[0, 0, 1000], bias=bias,
                buckets=buckets, cap=cap, seed=35, gap=1)
    assert p.plan(ctx).workspace_bytes(backward=True) > 4 * heads * 1801 + 100 * heads * buckets * 4 + 512
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_bad_values_in_ranges_of_the_backward_passes(ctx, precision):
    """A bad key, value and gradient reach the rows that see them, through every range's sum."""
    p = Problem([1100], [1100], 2, 1, 32, precision, mask=PREFIX, seed=36)
    p.k[900, 0, 3] = math.nan
    p.v[1000, 0, 1] = math.inf
    p.dout[800, 1, 2] = math.nan
    out = p.run(ctx)
    for n, rows in (("dq", 800), ("out", 900)):
        assert bool(torch.isfinite(out[n][:rows]).all()), n
    assert not bool(torch.isfinite(out["dq"][900:, 0]).any()) and not bool(torch.isfinite(out["dq"][800, 1]).any())
    assert bool(torch.isfinite(out["dq"][801:900]).all())


def test_too_many_tiles_are_refused(ctx):
    """Before anything is laid out for them."""
    n = 1 << 30
    with pytest.raises(gatgpu.GatGpuError) as err:
        gatgpu.Attention(ctx, [n] * 5, [n] * 5, heads=1, kv_heads=1, dim=32, precision=BF, q_begin=[i * n for i in range(5)],
                         k_begin=[i * n for i in range(5)])
    assert err.value.code == gatgpu.EOVERFLOW
