"""Cached attention in each of its forms (rows in tiles of 16, of 128 and of 256), where it can go wrong: against the plain form in 64 bits."""
import math

import pytest
import torch

import gatgpu
from cache_cases import EPS, Serving, generator, values, words

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
NONE = gatgpu.NO_PAGE
# Rows of a request that a call allows for, times the heads that share keys (two here), decide the form.
FORMS = [(FP, 16), (FP, 40), (FP, 400), (BF, 16), (BF, 40), (BF, 400)]
forms = pytest.mark.parametrize("precision,most", FORMS)
chunks = pytest.mark.parametrize("precision,most", [f for f in FORMS if f[1] > 16])


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def graph_of(ctx, calls):
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(ctx.stream())
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        calls()
    return graph


@chunks
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [16, 48, 80, 128])
def test_pages_and_widths(ctx, precision, most, page, dim):
    lens, rows = [1, 17, 64, 65, 300], [1, 17, 2, 9, 40]
    p = Serving(lens, rows, 4, 2, dim, page, precision, seed=dim + page, extra_rows=2, stride=3)
    p.check(p.run(ctx, most=most))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("heads,kv_heads,most", [(1, 1, 40), (1, 1, 200), (8, 1, 40), (6, 2, 12), (32, 1, 5), (64, 64, 33), (64, 1, 1), (40, 2, 20), (7, 7, 300)])
def test_heads(ctx, precision, heads, kv_heads, most):
    p = Serving([90, 20, 70], [min(most, 20), 1, 5 if most >= 5 else 1], heads, kv_heads, 32, 16, precision, seed=heads)
    p.check(p.run(ctx, most=most))


@forms
def test_rows_that_see_nothing(ctx, precision, most):
    """No tokens, fewer tokens than rows, tokens without pages, no rows."""
    p = Serving([0, 3, 40, 90, 50, 0], [2, 16, 0, 16, 3, 0], 4, 2, 64, 16, precision, seed=30)
    p.table[3] = [NONE] * len(p.table[3])
    p.table[4][0] = p.host.pages
    p.table[4][2] = 2 ** 31
    got = p.run(ctx, most=most)
    p.check(got)
    assert bool((got["lse"][:15] == -math.inf).all())


@forms
@pytest.mark.parametrize("page", [16, 64, 256])
def test_evicted_blocks_are_hidden(ctx, precision, most, page):
    p = Serving([11 * page + 7, 300], [16, 9], 4, 2, 64, page, precision, seed=31)
    for b in (0, 1, 5, 6, 7, 11):
        p.table[0][b] = NONE
    p.table[1][299 // page] = NONE  # the last block: the rows' own tokens
    p.check(p.run(ctx, most=most))


@forms
@pytest.mark.parametrize("value", [False, True])
def test_nan_reaches_the_rows_that_see_it(ctx, precision, most, value):
    """In the keys or the values of one token: the rows from its position on, of the heads that share it.  And in pages that nobody sees."""
    p = Serving([200, 90, 77], [16, 16, 16], 4, 2, 64, 16, precision, seed=32)
    for r, token, kv in ((0, 190, 1), (0, 199, 0), (1, 83, 0), (1, 5, 1), (2, 64, 0), (2, 63, 1)):
        data = p.host.sides()[1 if value else 0][0]
        data[p.table[r][token // 16], kv, token % 16, 7] = 0x7f if token % 2 else 0xff
    hidden = p.table[2][1]
    p.host.k[hidden], p.host.v[hidden] = 0x7f, 0xff
    p.table[2][1] = NONE
    p.check(p.run(ctx, most=most))


@forms
def test_bad_queries_stay_in_their_rows(ctx, precision, most):
    made = [Serving([100], [9], 4, 2, 32, 16, precision, seed=33) for _ in range(2)]
    q = made[0].q
    q[3, 1, 4], q[5, 2, 0], q[6, 0, 1] = math.nan, math.inf, -math.inf
    got, want = (p.run(ctx, most=most) for p in made)
    same = torch.ones(9, 4, dtype=torch.bool)
    same[3, 1] = same[5, 2] = same[6, 0] = False
    a, b = (x["out"].cpu()[:, :128].view(9, 4, 32) for x in (got, want))
    assert torch.equal(a[same], b[same]) and not bool(torch.isfinite(a[~same]).all())
    assert torch.equal(got["lse"].cpu()[same], want["lse"].cpu()[same])


@forms
def test_scales_far_apart(ctx, precision, most):
    """Pages whose values are 2^100 apart, scores of hundreds, and the least and the largest scales."""
    p = Serving([400, 400], [7, 16], 4, 2, 64, 16, precision, seed=34, size=8.0)
    g = generator(35)
    for r in range(2):
        for b in p.table[r]:
            if b != NONE:
                p.host.v_scale[b] = 2.0 ** torch.randint(-60, 41, (2,), generator=g).float()
    p.check(p.run(ctx, most=most))
    p = Serving([400], [5], 4, 2, 64, 16, precision, seed=36)
    for e in (-64, 64):
        p.host.v_scale[:] = 2.0 ** e
        p.check(p.run(ctx, most=most))


@forms
def test_work_cut_between_blocks(ctx, precision, most):
    """Requests of many tiles beside short ones: sums of several blocks are joined; equal calls give equal bits."""
    p = Serving([9000, 3, 1, 4097, 64, 130], [16, 1, 1, 9, 16, 0], 4, 2, 64, 32, precision, seed=37)
    got = p.run(ctx, most=most)
    p.check(got)
    again = p.run(ctx, most=most, lse=None)
    assert torch.equal(got["out"], again["out"]) and bool((again["lse"] == 7).all())


@chunks
@pytest.mark.parametrize("rows", [63, 64, 65, 129, 400])
def test_rows_at_the_ends_of_tiles(ctx, precision, most, rows):
    if rows > most:
        p = Serving([500], [rows], 4, 2, 32, 16, precision, seed=38)
        p.check(p.run(ctx, most=most), most=most)
        return
    p = Serving([500, rows], [rows, rows], 4, 2, 32, 16, precision, seed=38)
    p.check(p.run(ctx, most=most))


@forms
def test_only_the_first_rows_of_a_request(ctx, precision, most):
    p = Serving([60, 600], [most + 9, 4], 4, 2, 32, 16, precision, seed=39)
    p.check(p.run(ctx, most=most), most=most)


@chunks
@pytest.mark.parametrize("requests", [1023, 1025, 2100])
def test_many_requests(ctx, precision, most, requests):
    g = generator(requests)
    lens = torch.randint(1, 30, (requests,), generator=g).tolist()
    rows = [min(n, 1 + i % 3) if i % 5 else 0 for i, n in enumerate(lens)]
    lens[7], rows[7] = 200, 39
    p = Serving(lens, rows, 2, 1, 16, 16, precision, seed=40)
    p.check(p.run(ctx, most=most))


@forms
def test_lengths_and_offsets_beyond_their_arrays(ctx, precision, most):
    """Whatever the device arrays hold: no row beyond `rows`, no token beyond the table."""
    p = Serving([90, 80], [12, 4], 4, 2, 32, 16, precision, seed=41)
    d = p.device()
    d["lens"].copy_(words([2 ** 32 - 1, 80]))
    d["q_begin"].copy_(words([0, 12, 2 ** 31]))
    io = p.io(d, most=most)
    work = torch.empty(ctx.cache_attention_workspace(d["cache"], io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    p.k_len[0] = p.blocks * 16  # the same as all of the table
    p.check(d)
    d["q_begin"].copy_(words([16, 5, 0]))  # decreasing: no rows
    d["out"].fill_(7)
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    assert bool((d["out"] == 7).all())


@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("blocks", [0, 1, 64])
def test_no_token_in_the_table(ctx, most, blocks):
    """Tables of no blocks and of empty ones, and lengths that would not fit."""
    p = Serving([70, 1], [1, 1], 2, 1, 16, 16, BF, seed=42)
    p.table = [[NONE] * max(1, blocks) for _ in range(2)]
    d = p.device()
    io = p.io(d, most=most, blocks=blocks, table=d["table"].data_ptr() if blocks else None)
    work = torch.empty(ctx.cache_attention_workspace(d["cache"], io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    assert bool((d["out"][:2, :32] == 0).all()) and bool((d["lse"][:2] == -math.inf).all())


@pytest.mark.parametrize("kv_heads,most", [(4, 1), (8, 1), (2, 40)])
def test_as_many_requests_as_a_call_may_have(ctx, kv_heads, most):
    """2^20 requests, of which a few have a row; with 8 heads more threads than one launch takes if each had a block."""
    n, at = 2 ** 20, [0, 1, 4097, 2 ** 19, 2 ** 20 - 1]
    p = Serving([5, 33, 1, 64, 20], [1] * 5, kv_heads, kv_heads, 16, 16, BF, seed=43)
    d = p.device(gap=1)
    rows = torch.zeros(n, dtype=torch.int64)
    rows[at] = 1
    lens = torch.zeros(n, dtype=torch.int32)
    lens[at] = torch.tensor(p.k_len, dtype=torch.int32)
    table = torch.full((n, p.blocks), -1, dtype=torch.int32)
    table[at] = words([x for row in p.table for x in row]).cpu().view(5, -1)
    d.update(q_begin=torch.cat((torch.zeros(1, dtype=torch.int64), rows.cumsum(0))).int().cuda(), lens=lens.cuda(), table=table.cuda())
    io = p.io(d, requests=n, most=most)
    work = torch.empty(ctx.cache_attention_workspace(d["cache"], io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel())
    ctx.synchronize()
    p.check(d)


@forms
def test_captured_and_replayed(ctx, precision, most):
    """One graph, replayed over lengths and rows that change, with eager calls between."""
    shapes = [([600, 40, 70], [9, 16, 0]), ([601, 56, 71], [1, 16, 1]), ([1, 600, 0], [1, 1, 0]), ([600, 600, 600], [16, 1, 15])]
    made = [Serving(lens, rows, 4, 2, 64, 16, precision, seed=44 + i, extra_rows=32 - sum(rows)) for i, (lens, rows) in enumerate(shapes)]
    blocks, pages = max(p.blocks for p in made), max(p.host.pages for p in made)
    for p in made:  # of equal sizes
        p.table = [row + [NONE] * (blocks - len(row)) for row in p.table]
        p.blocks = blocks
        more = pages - p.host.pages
        for n in ("k", "v", "k_scale", "v_scale"):
            t = getattr(p.host, n)
            setattr(p.host, n, torch.cat((t, t[:1].expand(more, *t.shape[1:]))).contiguous())
        p.host.pages = pages
    d = made[0].device()
    io = made[0].io(d, most=most)
    work, other = (torch.empty(ctx.cache_attention_workspace(d["cache"], io), dtype=torch.uint8, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    graph = graph_of(ctx, lambda: ctx.cache_attention(d["cache"], io, work.data_ptr(), work.numel()))
    for p in made + made[:1]:
        e = p.device()
        for n in ("k", "v", "k_scale", "v_scale", "q", "q_begin", "lens", "table", "out", "lse"):
            d[n].copy_(e[n])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.check(d)
        ctx.cache_attention(e["cache"], p.io(e, most=most), other.data_ptr(), other.numel())
        ctx.synchronize()
        assert torch.equal(e["out"], d["out"]) and torch.equal(e["lse"], d["lse"])


@pytest.mark.parametrize("most", [16, 40, 400])
def test_two_contexts_at_once(ctx, most):
    """Calls in flight of two contexts, a workspace each."""
    made = [Serving([5000, 70], [3, 9], 4, 2, 64, 16, BF, seed=s) for s in (50, 51)]
    want = [p.run(ctx, most=most)["out"] for p in made]
    with gatgpu.Context(0) as second:
        held = [(c, p, p.device(gap=1)) for c, p in zip((ctx, second), made)]
        work = [torch.empty(c.cache_attention_workspace(d["cache"], p.io(d, most=most)), dtype=torch.uint8, device="cuda") for c, p, d in held]
        torch.cuda.synchronize()
        for _ in range(5):
            for (c, p, d), w in zip(held, work):
                c.cache_attention(d["cache"], p.io(d, most=most), w.data_ptr(), w.numel())
        torch.cuda.synchronize()
    for (_, _, d), x in zip(held, want):
        assert torch.equal(d["out"], x)


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("requests,kv_heads,group,rows,most_keys", [(150, 1, 2, 1, 3000), (70, 4, 4, 16, 1500), (70, 4, 2, 16, 1500), (200, 2, 8, 2, 1500)])
def test_ranges_over_many_requests(ctx, precision, requests, kv_heads, group, rows, most_keys):
    """A block's range ends in one request and goes on in others, of one to four row tiles side by side."""
    g = generator(requests + group)
    lens = torch.randint(1, most_keys // 8, (requests,), generator=g).tolist()
    lens[3], lens[40], lens[requests - 1] = most_keys, most_keys - 1, 0
    q_len = [int(torch.randint(0, min(rows, n) + 1, (1,), generator=g)) for n in lens]
    q_len[3], q_len[40] = rows, rows
    p = Serving(lens, q_len, kv_heads * group, kv_heads, 16, 16, precision, seed=requests)
    p.check(p.run(ctx))


@pytest.mark.parametrize("precision", [FP, BF])
@pytest.mark.parametrize("group,rows,lens", [(1, 1, [41_000, 3000]), (4, 16, [9000, 5000, 64]), (3, 15, [14_000, 130, 0]), (2, 13, [4100, 4097, 33, 700]), (4, 8, [1100, 90])])
def test_ranges_of_few_requests(ctx, precision, group, rows, lens):
    """One to four row tiles side by side, ranges that end between the key tiles of some and of others, in every amount of work."""
    q_len = [min(rows - i, n) for i, n in enumerate(lens)]
    p = Serving(lens, [max(0, n) for n in q_len], 8 * group, 8, 16, 16, precision, seed=60 + rows)
    p.check(p.run(ctx))


@pytest.mark.parametrize("keys", [511, 512, 513, 1023, 1024, 1025])
@forms
def test_where_a_block_takes_a_row_tile_alone(ctx, precision, most, keys):
    """Tables at the lengths where the forms change, and one whose blocks are too many for that."""
    p = Serving([keys, 90], [16, 16], 4, 2, 16, 16, precision, seed=keys)
    p.check(p.run(ctx, most=most))
    if keys == 512:
        p = Serving([keys] + [20] * 300, [16] + [1] * 300, 4, 2, 16, 16, precision, seed=keys)
        p.check(p.run(ctx, most=most))
        p.check(p.run(ctx, most=5000))


@forms
@pytest.mark.parametrize("size", [1e5, 3e7, 1e9, 1e12, 1e30])
def test_far_scores(ctx, precision, most, size):
    """Scores whose steps in FP32 are wider than the room between a weight and its reference: the largest one's value, of either sign."""
    p = Serving([70, 300], [16, 16], 4, 2, 32, 16, precision, seed=70)
    for side in (p.host.k, p.host.k_scale):
        side.zero_()
    for r, keys in enumerate(p.k_len):
        for t in range(keys):
            page = p.table[r][t // 16]
            p.host.k[page, :, t % 16] = 0xb8  # -1, and 1 in one column
            p.host.k[page, :, t % 16, t * 7 % 31] = 0x38
    p.host.k_scale[:] = 1.0
    hot = [(3, 1, 0), (9, 2, 12), (20, 0, 30), (31, 3, 5)]  # row, head, column: 1 there, and 0 elsewhere
    for row, head, c in hot:
        p.q[row, head] = 0
        p.q[row, head, c] = size
    p.q[11] *= size
    p.q[14] *= -size
    p.q[25] = -size  # every score is size 30 but for rounding
    d = p.run(ctx, most=most)
    p.check(d)
    out, lse = d["out"].cpu()[:, :128].view(32, 4, 32).double(), d["lse"].cpu().double()
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    for row, head, c in hot:
        r, i = divmod(row, 16)
        seen = p.k_len[r] - 16 + i + 1
        kv = head // 2
        them = [t for t in range(seen) if t * 7 % 31 == c]
        if not them:
            continue
        v = torch.stack([values(p.host.v[p.table[r][t // 16], kv, :, t % 16]) * float(p.host.v_scale[p.table[r][t // 16], kv]) for t in them])
        # (equal scores: their mean; the weights and their sum are exact but for 2^-21, and fp16's rounding where it is no power of two)
        tol = v.abs().mean(0) * (2.0 ** -20 + (2.0 ** -11 if precision == BF else 2.0 ** -22)) + v.mean(0).abs() * EPS[precision]
        assert bool(((out[row, head] - v.mean(0)).abs() <= tol).all())
        top = p.scale * float(p.q[row, head, c])
        assert abs(float(lse[row, head]) - top - math.log(len(them))) <= top * 2.0 ** -21


@forms
@pytest.mark.parametrize("scale", [1e-40, 1e-30, 1e30])
def test_scales_beyond_reason(ctx, precision, most, scale):
    """Factors of scores that would leave FP32: what is not seen stays so, scores of 0 stay 0."""
    p = Serving([90, 200], [16, 16], 4, 2, 32, 16, precision, seed=71)
    for s in (p.host.k_scale, p.host.v_scale):
        s[:] = 2.0 ** -64 if scale < 1 else 2.0 ** 64
    p.host.v_scale[:] = 1.0
    if scale > 1:
        p.q.zero_()
    p.table[0][2] = NONE
    p.scale = scale
    p.check(p.run(ctx, most=most))
