"""The paged 8-bit cache on the GPU: what append writes and what attention reads, against plain forms in 64 bits."""
import math

import numpy as np
import pytest
import torch

import gatgpu
from cache_cases import TYPE, Pages, Serving, generator, normal, words

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
NONE = gatgpu.NO_PAGE


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def append(ctx, d, k, v, slots, precision, gap=0):
    """Rows of keys and values side by side, `gap` chunks behind them."""
    rows, heads, dim = k.shape
    per = 8 if precision == BF else 4
    kv = torch.full((max(1, rows), 2 * heads * dim + gap * per), math.nan, dtype=TYPE[precision])
    kv[:rows, :heads * dim] = k.reshape(rows, heads * dim)
    kv[:rows, heads * dim:2 * heads * dim] = v.reshape(rows, heads * dim)
    kv, slot = kv.cuda(), words(slots) if rows else words([0])
    io = gatgpu.AppendIO(precision=precision, rows=rows, k=kv.data_ptr(), v=kv.data_ptr() + heads * dim * kv.element_size(), k_stride=kv.stride(0),
                         v_stride=kv.stride(0), slot=slot.data_ptr())
    torch.cuda.synchronize()
    ctx.cache_append(d["cache"], io)
    ctx.synchronize()


def rows_of(g, n, heads, dim, precision, size=1.0):
    return [(normal(g, n, heads, dim) * size).to(TYPE[precision]) for _ in range(2)]


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim,heads", [(16, 1), (48, 3), (64, 2), (128, 2)])
def test_append_whole_and_open_pages(ctx, precision, page, dim, heads):
    """A prompt that begins and ends within pages, then token by token, with values that grow and shrink."""
    g = generator(page + dim)
    host = Pages(9, page, heads, dim, seed=1)
    d = host.device()
    order = torch.randperm(9, generator=g).tolist()
    slots = [order[t // page] * page + t % page for t in range(9 * page)]
    at = 0
    for n, size in ((page // 2 + 3, 1.0), (3 * page, 5.0), (1, 0.1), (1, 40.0), (1, 3000.0), (5, 1e-3), (page, 1.0), (2 * page, 0.02)):
        k, v = rows_of(g, n, heads, dim, precision, size)
        host.append(k, v, torch.tensor(slots[at:at + n]))
        append(ctx, d, k, v, slots[at:at + n], precision, gap=1)
        host.same_values(d)
        at += n


@pytest.mark.parametrize("precision", [FP, BF])
def test_append_tokens_of_many_requests(ctx, precision):
    """One token each of requests at any offset, rows without a slot between them; and more rows than the kernel takes singly."""
    g = generator(2)
    for runs, most in ((90, 1), (700, 9), (4200, 1), (1500, 7)):
        host = Pages(runs + 10, 16, 2, 32, seed=3)
        d = host.device()
        slots = []
        for p in torch.randperm(runs + 10, generator=g).tolist()[:runs]:  # one to `most` tokens from any offset on
            n, off = int(torch.randint(1, most + 1, (1,), generator=g)), int(torch.randint(0, 16, (1,), generator=g))
            slots += [p * 16 + o for o in range(off, min(16, off + n))]
        rows = len(slots)
        bad = (NONE, (runs + 10) * 16, 2 ** 31, NONE)
        for j, i in enumerate(range(0, rows, 11)):
            if i + 1 == rows or slots[i + 1] != slots[i] + 1:  # (a gap within a page's tokens is none of the operator's)
                slots[i] = bad[j % 4]
        k, v = rows_of(g, rows, 2, 32, precision)
        host.append(k, v, torch.tensor(slots))
        append(ctx, d, k, v, slots, precision)
        host.same_values(d)


@pytest.mark.parametrize("precision", [FP, BF])
def test_append_values_of_every_size(ctx, precision):
    """Zeros, the least and the largest values, ties, NaN and infinities."""
    host = Pages(8, 16, 1, 16, seed=4)
    d = host.device()
    t = TYPE[precision]
    k, v = torch.zeros(8 * 16, 1, 16, dtype=t), torch.ones(8 * 16, 1, 16, dtype=t)
    k[16:32] = 1e-30
    k[32:48, 0, 3] = 3e38
    k[32:48, 0, 4] = -1e-38
    k[48, 0, 0], k[49, 0, 1], k[50, 0, 2], k[51, 0, 3] = math.nan, math.inf, -math.inf, 2.0
    k[64:80] = (448.0 * 2.0 ** torch.arange(-8, 8).float()).view(16, 1, 1).to(t)
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    between = torch.cat((every, (every[1:] + every[:-1]) / 2, torch.tensor([448.0, 2.0 ** -10, 3 * 2.0 ** -10])))[:256]
    v[80:96, 0] = between.view(16, 16).to(t)
    v[96:112] = math.nan
    v[112:, 0, 5] = -math.inf
    host.append(k, v, torch.arange(128))
    append(ctx, d, k, v, list(range(128)), precision)
    host.same_values(d)
    assert float(d["k_scale"][0, 0]) == 2.0 ** -64 and float(d["k_scale"][2, 0]) == 2.0 ** 64 and float(d["v_scale"][6, 0]) == 2.0 ** -64


def test_append_scale_grows_from_the_least_to_the_largest(ctx):
    host = Pages(2, 16, 1, 32, seed=5)
    d = host.device()
    g = generator(6)
    for t in range(16):
        k, v = rows_of(g, 1, 1, 32, FP, 10.0 ** (-20 + 2.5 * t))
        host.append(k, v, torch.tensor([16 + t]))
        append(ctx, d, k, v, [16 + t], FP)
        host.same_values(d)


def test_append_writes_the_pages_of_the_slots_only(ctx):
    host = Pages(6, 32, 2, 64, seed=7)
    d = host.device()
    k, v = rows_of(generator(8), 40, 2, 64, BF)
    before = {n: d[n].clone() for n in ("k", "v")}
    append(ctx, d, k, v, list(range(70, 110)), BF)  # pages 2 and 3, the first from token 6 on
    for n in ("k", "v"):
        same = d[n] == before[n]
        assert bool(same[[0, 1, 4, 5]].all())
    assert torch.equal(d["k"][3, :, 14:], before["k"][3, :, 14:]) and torch.equal(d["v"][3, :, :, 14:], before["v"][3, :, :, 14:])
    append(ctx, d, k[:0], v[:0], [], BF)  # no rows


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128])
def test_one_token_each(ctx, precision, page, dim):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 700]
    p = Serving(lens, [1] * len(lens), 4, 2, dim, page, precision, seed=dim + page, extra_rows=2, stride=3)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (6, 2), (32, 1), (5, 5), (14, 2), (40, 2)])
@pytest.mark.parametrize("q_len", [1, 3, 20])
def test_shared_heads_and_rows(ctx, precision, heads, kv_heads, q_len):
    p = Serving([130, 20, 77], [q_len, min(q_len, 20), 1], heads, kv_heads, 32, 16, precision, seed=heads)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (96, 32)])
def test_chunks_of_prompts(ctx, precision, dim, page):
    """Many rows of a request, over tokens before them and from the beginning."""
    p = Serving([300, 129, 64, 500], [200, 129, 1, 33], 4, 2, dim, page, precision, seed=dim)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_long_and_short_requests_together(ctx, precision):
    p = Serving([9000, 3, 1, 4097, 64, 130], [1, 1, 1, 2, 1, 1], 8, 4, 64, 32, precision, seed=9)
    p.check(p.run(ctx))


def test_one_request_over_the_whole_chip(ctx):
    p = Serving([70_001], [1], 2, 1, 128, 64, BF, seed=10)
    p.check(p.run(ctx))


@pytest.mark.parametrize("requests", [255, 256, 257, 1100])
def test_many_requests(ctx, requests):
    rng = np.random.default_rng(requests)
    lens = rng.integers(1, 40, requests).tolist()
    p = Serving(lens, [1] * requests, 2, 1, 16, 16, BF, seed=11)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_rows_that_see_nothing(ctx, precision):
    """No tokens, fewer tokens than rows, tokens without pages, no rows."""
    p = Serving([0, 3, 40, 90, 50, 0], [2, 7, 0, 1, 3, 0], 4, 2, 64, 16, precision, seed=12)
    p.table[3] = [NONE] * len(p.table[3])
    p.table[4][0] = p.host.pages
    p.table[4][2] = 2 ** 31
    got = p.run(ctx)
    p.check(got)
    assert bool((got["lse"][:6] == -math.inf).all())


@pytest.mark.parametrize("precision", [FP, BF])
def test_evicted_blocks_are_hidden(ctx, precision):
    p = Serving([700, 300], [3, 1], 4, 2, 64, 32, precision, seed=13)
    for b in (0, 1, 5, 6, 7, 20):
        p.table[0][b] = NONE
    p.table[1][9] = NONE  # the last block: its own token among it
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("value", [False, True])
def test_nan_reaches_the_rows_that_see_it(ctx, precision, value):
    """In the keys or the values of one token: the rows from its position on, of the heads that share it."""
    p = Serving([200, 90], [60, 60], 4, 2, 64, 16, precision, seed=14)
    for r, token, kv in ((0, 170, 1), (0, 199, 0), (1, 33, 0), (1, 5, 1)):
        data = p.host.sides()[1 if value else 0][0]
        data[p.table[r][token // 16], kv, token % 16, 7] = 0x7f if token % 2 else 0xff
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
def test_bad_queries_stay_in_their_rows(ctx, precision):
    p = Serving([100], [9], 4, 2, 32, 16, precision, seed=15)
    p.q[3, 1, 4], p.q[5, 2, 0], p.q[6, 0, 1] = math.nan, math.inf, -math.inf
    d = p.run(ctx)
    want = Serving([100], [9], 4, 2, 32, 16, precision, seed=15)
    other = want.run(ctx)
    same = torch.ones(9, 4, dtype=torch.bool)
    same[3, 1] = same[5, 2] = same[6, 0] = False
    a, b = (x["out"].cpu()[:, :128].view(9, 4, 32) for x in (d, other))
    assert torch.equal(a[same], b[same]) and not bool(torch.isfinite(a[~same]).all())
    assert torch.equal(d["lse"].cpu()[same], other["lse"].cpu()[same])


@pytest.mark.parametrize("precision", [FP, BF])
def test_scales_far_apart(ctx, precision):
    """Pages whose values are 2^100 apart: the weights decide, not the pages' sizes; and scores of hundreds."""
    p = Serving([400, 400], [1, 2], 4, 2, 64, 16, precision, seed=16, size=8.0)
    g = generator(17)
    for r in range(2):
        for b in p.table[r]:
            if b != NONE:
                p.host.v_scale[b] = 2.0 ** torch.randint(-60, 41, (2,), generator=g).float()
    p.check(p.run(ctx))
    p = Serving([400], [1], 4, 2, 64, 16, precision, seed=18)
    p.host.v_scale[:] = 2.0 ** -64
    p.check(p.run(ctx))
    p.host.v_scale[:] = 2.0 ** 64
    p.check(p.run(ctx))


def test_only_the_first_rows_of_a_request(ctx):
    p = Serving([50, 60], [9, 4], 4, 2, 32, 16, BF, seed=19)
    p.check(p.run(ctx, most=3), most=3)


def test_lse_may_be_left_out_and_bits_are_equal(ctx):
    p = Serving([3000, 50], [1, 1], 8, 2, 64, 16, BF, seed=20)
    a, b = p.run(ctx), p.run(ctx, lse=None)
    assert torch.equal(a["out"], b["out"]) and bool((b["lse"] == 7).all())


def test_lengths_and_offsets_beyond_their_arrays(ctx):
    """Whatever the device arrays hold: no row beyond `rows`, no token beyond the table."""
    p = Serving([90, 80], [1, 1], 2, 1, 32, 16, BF, seed=21)
    d = p.device()
    d["lens"].copy_(words([2 ** 32 - 1, 80]))
    d["q_begin"].copy_(words([0, 1, 2 ** 31]))
    io = p.io(d)
    work = torch.empty(ctx.cache_attention_workspace(d["cache"], io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    p.k_len[0] = p.blocks * 16  # the same as all of the table
    p.check(d)
    d["q_begin"].copy_(words([5, 1, 0]))  # decreasing: no rows
    d["out"].fill_(7)
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    assert bool((d["out"] == 7).all())


def test_refusals(ctx):
    p = Serving([20, 30], [1, 2], 4, 2, 32, 16, BF, seed=22)
    d = p.device()
    work = torch.empty(ctx.cache_attention_workspace(d["cache"], p.io(d)), dtype=torch.uint8, device="cuda")

    def cache(**change):
        c = gatgpu.Cache.from_buffer_copy(d["cache"])
        for k, v in change.items():
            setattr(c, k, v)
        return c

    def refused(code=gatgpu.EINVAL, c=None, ws=work.data_ptr(), size=work.numel(), **change):
        with pytest.raises(gatgpu.GatGpuError) as err:
            ctx.cache_attention(c or d["cache"], p.io(d, **change), ws, size)
        assert err.value.code == code, str(err.value)

    bad = [dict(page=8), dict(page=20), dict(page=512), dict(pages=0), dict(kv_heads=0), dict(kv_heads=65), dict(dim=8), dict(dim=24), dict(dim=144),
           dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=d["k"].data_ptr() + 8), dict(v_scale=np.zeros(8).ctypes.data // 16 * 16)]
    for change in bad:
        refused(c=cache(**change))
        with pytest.raises(gatgpu.GatGpuError):
            ctx.cache_append(cache(**change), gatgpu.AppendIO(precision=BF))
    refused(gatgpu.EOVERFLOW, c=cache(pages=2 ** 28))
    for change in (dict(precision=2), dict(heads=3), dict(heads=0), dict(heads=66), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=None),
                   dict(out=None), dict(q_begin=None), dict(k_len=None), dict(table=None), dict(q_stride=127), dict(out_stride=2 ** 45),
                   dict(q=d["q"].data_ptr() + 4), dict(out_stride=p.io(d).out_stride + 1), dict(table_stride=1), dict(lse=d["lse"].data_ptr() + 1),
                   dict(k_len=np.zeros(4, np.uint32).ctypes.data)):
        refused(**change)
    refused(gatgpu.EOVERFLOW, rows=2 ** 29)
    refused(gatgpu.EOVERFLOW, requests=2 ** 20 + 1)
    refused(gatgpu.EOVERFLOW, blocks=2 ** 28, table_stride=2 ** 28)
    refused(ws=None)
    refused(ws=work.data_ptr() + 8)
    refused(size=work.numel() - 1)
    with pytest.raises(gatgpu.GatGpuError):
        ctx.cache_attention(None, p.io(d))
    for io in (gatgpu.AppendIO(precision=3), gatgpu.AppendIO(precision=BF, rows=1), None,
               gatgpu.AppendIO(precision=BF, rows=1, k=d["q"].data_ptr(), v=d["q"].data_ptr(), k_stride=64, v_stride=64),
               gatgpu.AppendIO(precision=BF, rows=1, k=d["q"].data_ptr(), v=d["q"].data_ptr(), k_stride=63, v_stride=64, slot=d["lens"].data_ptr()),
               gatgpu.AppendIO(precision=BF, rows=2 ** 27, k=d["q"].data_ptr(), v=d["q"].data_ptr(), k_stride=64, v_stride=64, slot=d["lens"].data_ptr())):
        with pytest.raises(gatgpu.GatGpuError):
            ctx.cache_append(d["cache"], io)
    ctx.cache_attention(d["cache"], p.io(d, requests=0))  # nothing to do: no workspace needed
    ctx.cache_attention(d["cache"], p.io(d, rows=0, q=None))
