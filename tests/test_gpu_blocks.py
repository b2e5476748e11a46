"""Block tables, slots and free lists on the GPU against one request after another."""
import numpy as np
import pytest
import torch

import gatgpu
from cache_cases import assign, release

pytestmark = pytest.mark.gpu

NONE = gatgpu.NO_PAGE
OUTPUTS = ("stored", "k_len", "q_begin", "slot", "position", "free_left", "unserved")


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def words(values, n=None):
    a = np.asarray(list(values), np.uint64).astype(np.uint32)
    return torch.from_numpy(np.concatenate((a, np.zeros((n or a.size) - a.size, np.uint32))).view(np.int32)).cuda()


def back(t):
    return t.cpu().numpy().view(np.uint32)


class Problem:
    def __init__(self, cached, fresh, page=16, blocks=None, spare=None, rows=None, seed=0, stride=0):
        rng = np.random.default_rng(seed)
        self.cached, self.fresh, self.page = list(cached), list(fresh), page
        held = [-(-c // page) for c in self.cached]
        total = [-(-(c + f) // page) for c, f in zip(self.cached, self.fresh)]
        self.blocks = max(total + held + [1]) if blocks is None else blocks
        need = sum(total) - sum(held)
        self.count = need + 2 if spare is None else spare
        self.pages = sum(held) + max(need, self.count) + 3
        self.rows = sum(self.fresh) + 5 if rows is None else rows
        order = rng.permutation(self.pages).tolist()
        self.stride = self.blocks + stride
        self.table = [[NONE] * self.stride for _ in self.cached]
        for r, h in enumerate(held):
            for b in range(min(h, self.blocks)):
                self.table[r][b] = order.pop()
        self.free = [order.pop() for _ in range(min(self.count, len(order)))]
        self.free += [NONE] * (self.pages - len(self.free))

    def io(self, d, **change):
        io = gatgpu.BlocksIO(requests=len(self.cached), page=self.page, pages=self.pages, rows=self.rows, blocks=self.blocks, table_stride=self.stride,
                             **{n: t.data_ptr() for n, t in d.items()})
        for k, v in change.items():
            setattr(io, k, v)
        return io

    def device(self):
        n = len(self.cached)
        d = {"cached": words(self.cached, max(1, n)), "fresh": words(self.fresh, max(1, n)), "free": words(self.free), "free_count": words([self.count]),
             "table": words([x for row in self.table for x in row], max(1, n * self.stride))}
        for name, size in (("free_left", 1), ("stored", n), ("k_len", n), ("q_begin", n + 1), ("slot", self.rows), ("position", self.rows), ("unserved", 1)):
            d[name] = torch.full((max(1, size),), 77, dtype=torch.int32, device="cuda")
        return d

    def run(self, ctx, in_place=False, d=None):
        d = self.device() if d is None else d
        if in_place:
            d["stored"], d["free_left"] = d["cached"], d["free_count"]
        io = self.io(d)
        need = ctx.blocks_workspace(io)
        work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        ctx.blocks_assign(io, work.data_ptr(), need)
        ctx.synchronize()
        return d

    def check(self, d):
        table = [row[:] for row in self.table]
        want = assign(self.cached, self.fresh, table, self.free, self.count, self.page, self.pages, self.blocks, self.rows)
        for name in OUTPUTS:
            got = back(d[name])[:len(want[name])].tolist()
            assert got == want[name], (name, [(i, a, b) for i, (a, b) in enumerate(zip(got, want[name])) if a != b][:5])
        assert back(d["table"])[:len(table) * self.stride].tolist() == [x for row in table for x in row]
        assert back(d["free"]).tolist() == self.free
        return want


def lengths(n, most, seed, some=True):
    rng = np.random.default_rng(seed)
    return [int(x) * int(rng.integers(0, 2) if some else 1) for x in rng.integers(1, most + 1, n)]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("requests,cached,fresh", [(1, 0, 1), (1, 300, 40), (12, 100, 1), (40, 300, 70), (1000, 40, 5), (1000, 9, 30), (1025, 50, 3), (4097, 30, 30), (64, 90, 32), (64, 90, 33)])
def test_steps(ctx, page, requests, cached, fresh):
    p = Problem(lengths(requests, cached, 1) if cached else [0] * requests, lengths(requests, fresh, 2, some=requests > 12), page, seed=requests, stride=3)
    p.check(p.run(ctx))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,rows", [(30, None), (30, 9000), (1500, None)])
def test_in_place(ctx, in_place, requests, rows):
    p = Problem(lengths(requests, 60, 3), lengths(requests, 20, 4), rows=rows, seed=5)
    d = p.run(ctx, in_place=in_place)
    p.check(d)


@pytest.mark.parametrize("requests", [20, 1200])
def test_too_few_pages_rows_or_blocks(ctx, requests):
    c, f = lengths(requests, 60, 6), lengths(requests, 40, 7)
    for spare in (0, 1, 17):
        want = Problem(c, f, spare=spare, seed=8)
        assert want.check(want.run(ctx))["unserved"][0] > 0
    p = Problem(c, f, rows=sum(f) // 2, seed=9)
    assert p.check(p.run(ctx))["unserved"][0] > 0
    p = Problem(c, f, blocks=4, seed=10)
    assert p.check(p.run(ctx))["unserved"][0] > 0
    p = Problem(c, f, rows=0, seed=11)
    p.check(p.run(ctx))


def test_no_requests_and_empty_ones(ctx):
    p = Problem([], [], rows=40)
    p.check(p.run(ctx))
    p = Problem([0, 5, 0, 16, 0], [0, 0, 0, 0, 0], rows=3)
    p.check(p.run(ctx))
    p = Problem([0, 5, 0, 16, 0], [0, 11, 0, 16, 33], rows=9000)  # two launches
    p.check(p.run(ctx))


def test_lengths_that_wrap(ctx):
    """Lengths and sums of lengths beyond 32 bits are not served; nothing is written for them."""
    p = Problem([5, 0, 7], [3, 4, 2], blocks=4, seed=12)
    p.cached[0], p.fresh[1] = 2 ** 32 - 1, 2 ** 32 - 1
    p.check(p.run(ctx))
    p.fresh[2] = 2 ** 32 - 1
    p.check(p.run(ctx))


@pytest.mark.parametrize("rows", [60, 9000])
def test_bad_pages_and_counts(ctx, rows):
    """Entries that are no pages give rows without slots; a count beyond the list is the list."""
    p = Problem([20, 40, 3], [5, 20, 30], rows=rows, seed=13)
    p.table[0][1] = p.pages
    p.table[1][2] = NONE
    p.free[p.count - 1] = 2 ** 31
    p.check(p.run(ctx))
    p = Problem([20, 40, 3], [5, 20, 30], rows=rows, seed=13)
    p.free = [int(x) for x in np.random.default_rng(1).permutation(p.pages)]
    p.count = 2 ** 32 - 1
    p.check(p.run(ctx))


@pytest.mark.parametrize("requests", [1, 7, 32, 33, 65, 2000, 20_000, 33_000])
@pytest.mark.parametrize("in_place", [False, True])
def test_release(ctx, requests, in_place):
    p = Problem(lengths(requests, 400 if requests < 5000 else 40, 14), [0] * requests, seed=15, stride=2)
    rng = np.random.default_rng(16)
    for r in range(0, requests, 3):  # pages that were given up before
        if p.cached[r]:
            p.table[r][rng.integers(0, -(-p.cached[r] // p.page))] = NONE
    d = p.device()
    if in_place:
        d["free_left"] = d["free_count"]
    io = p.io(d)
    need = ctx.blocks_workspace(io)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.blocks_release(io, work.data_ptr(), need)
    ctx.synchronize()
    free = p.free[:]
    left = release(p.cached, p.table, free, p.count, p.page, p.pages, p.blocks)
    assert back(d["free"]).tolist() == free and back(d["free_left"]).tolist() == [left]
    assert back(d["table"]).tolist()[:requests * p.stride] == [x for row in p.table for x in row]


@pytest.mark.parametrize("requests", [50, 600])
def test_release_beyond_the_list(ctx, requests):
    """Pages given back twice: what the list has no place for is dropped."""
    p = Problem([100] * requests, [0] * requests, blocks=5, seed=17)
    p.count = p.pages - 4
    p.free = [0] * p.pages
    d = p.device()
    io = p.io(d)
    need = ctx.blocks_workspace(io)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.blocks_release(io, work.data_ptr(), need)
    ctx.synchronize()
    free = p.free[:]
    assert release(p.cached, p.table, free, p.count, p.page, p.pages, p.blocks) == p.pages == back(d["free_left"])[0]
    assert back(d["free"]).tolist() == free


def test_captured_steps_run_on(ctx):
    """A captured decoding step, replayed: each goes on from the lengths and the list that the one before left."""
    n = 9
    p = Problem(lengths(n, 60, 18), [1] * n, spare=40, seed=19)
    p.blocks = p.stride = 10
    for row in p.table:
        row += [NONE] * (10 - len(row))
    d = p.device()
    d["stored"], d["free_left"] = d["cached"], d["free_count"]
    io = p.io(d)
    work = torch.empty(ctx.blocks_workspace(io), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(ctx.stream())
    with torch.cuda.graph(graph, stream=stream):
        ctx.blocks_assign(io, work.data_ptr(), work.numel())
    for i in range(30):
        if i == 20:  # fewer requests go on
            d["fresh"][::2] = 0
            p.fresh = [0 if r % 2 == 0 else 1 for r in range(n)]
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = p.check(d)
        p.cached, p.count = want["stored"], want["free_left"][0]
        p.table = back(d["table"]).reshape(n, 10).tolist()


def test_refusals(ctx):
    p = Problem([3, 4], [1, 2])
    d = p.device()
    work = torch.empty(4096, dtype=torch.uint8, device="cuda")

    def refused(call=ctx.blocks_assign, code=gatgpu.EINVAL, ws=work.data_ptr(), size=4096, **change):
        with pytest.raises(gatgpu.GatGpuError) as err:
            call(p.io(d, **change), ws, size)
        assert err.value.code == code, str(err.value)

    for call in (ctx.blocks_assign, ctx.blocks_release):
        for change in (dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(table_stride=p.blocks - 1), dict(table_stride=2 ** 41), dict(cached=None),
                       dict(table=None), dict(free=None), dict(free_count=None), dict(free_left=None), dict(free=d["free"].data_ptr() + 2),
                       dict(cached=np.zeros(4, np.uint32).ctypes.data)):
            refused(call, **change)
        refused(call, gatgpu.EOVERFLOW, requests=2 ** 20 + 1)
        refused(call, gatgpu.EOVERFLOW, pages=2 ** 28)
        refused(call, gatgpu.EOVERFLOW, blocks=2 ** 28, table_stride=2 ** 28)
        refused(call, ws=None)
        refused(call, ws=work.data_ptr() + 8)
        refused(call, size=8)
    for name in ("fresh", "stored", "k_len", "q_begin", "slot", "position", "unserved"):
        refused(**{name: None})
