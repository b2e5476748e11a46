"""The operators together, as they are used: steps of a server over a paged cache, captured and replayed, and a layer that trains."""
import math

import numpy as np
import pytest
import torch

import gatgpu
from attention_cases import Problem as AttentionProblem
from cache_cases import TYPE, Pages, assign, check_attention, generator, normal, release, rotate, rotate_bound, words
from test_gpu_rotate import Problem as RotateProblem

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
HALVES, NEIGHBOURS = gatgpu.PAIRS_HALVES, gatgpu.PAIRS_NEIGHBOURS
NONE = gatgpu.NO_PAGE


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def host(t):
    return t.cpu().numpy().view(np.uint32)


class Server:
    """Requests of a fixed batch; everything a step reads or writes has its place for good, so that a step is one graph."""

    def __init__(self, ctx, precision, requests, rows, most, page, pages, blocks, heads, kv_heads, dim, pairs, seed=0):
        self.ctx, self.precision, self.requests, self.rows, self.most = ctx, precision, requests, rows, most
        self.page, self.pages, self.blocks, self.heads, self.kv_heads, self.dim, self.pairs = page, pages, blocks, heads, kv_heads, dim, pairs
        self.eps, self.rot, self.scale = 1e-6, dim, dim ** -0.5
        self.g = generator(seed)
        t = TYPE[precision]
        self.width = (heads + 2 * kv_heads) * dim
        self.gamma = [1 + 0.2 * normal(self.g, dim) for _ in range(2)]
        self.freq = torch.pow(1e4, -2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
        # The host's copy of the state.
        self.host = Pages(pages, page, kv_heads, dim, seed=seed + 1)
        self.cached, self.table = [0] * requests, [[NONE] * blocks for _ in range(requests)]
        order = torch.randperm(pages, generator=self.g).tolist()
        self.free, self.count = order, pages
        # The device's.
        d = self.d = self.host.device()
        zero = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        d.update(cached=zero(requests), fresh=zero(requests), gone=zero(requests), free=words(order), free_count=words([pages]),
                 table=words([x for row in self.table for x in row]), k_len=zero(requests), q_begin=zero(requests + 1), slot=zero(rows), position=zero(rows),
                 unserved=zero(1), qkv=torch.zeros(rows, self.width, dtype=t, device="cuda"), turned=torch.zeros(rows, self.width, dtype=t, device="cuda"),
                 out=torch.zeros(rows, heads * dim, dtype=t, device="cuda"), lse=torch.zeros(rows, heads, device="cuda"),
                 gamma=[x.cuda() for x in self.gamma], freq_=self.freq.cuda())
        size, at, v = d["qkv"].element_size(), heads * dim, (heads + kv_heads) * dim
        self.blocks_io = gatgpu.BlocksIO(requests=requests, page=page, pages=pages, rows=rows, blocks=blocks, table_stride=blocks,
                                         **{n: d[n].data_ptr() for n in ("cached", "fresh", "table", "free", "free_count", "k_len", "q_begin", "slot", "position", "unserved")},
                                         free_left=d["free_count"].data_ptr(), stored=d["cached"].data_ptr())
        self.release_io = gatgpu.BlocksIO(requests=requests, page=page, pages=pages, blocks=blocks, table_stride=blocks, cached=d["gone"].data_ptr(),
                                          table=d["table"].data_ptr(), free=d["free"].data_ptr(), free_count=d["free_count"].data_ptr(), free_left=d["free_count"].data_ptr())
        self.rotate_io = gatgpu.RotateIO(precision=precision, heads=heads, kv_heads=kv_heads, dim=dim, norm=1, rot=self.rot, pairs=pairs, eps=self.eps, rows=rows,
                                         q=d["qkv"].data_ptr(), k=d["qkv"].data_ptr() + at * size, q_stride=self.width, k_stride=self.width,
                                         gamma_q=d["gamma"][0].data_ptr(), gamma_k=d["gamma"][1].data_ptr(), position=d["position"].data_ptr(),
                                         freq=d["freq_"].data_ptr(), q_out=d["turned"].data_ptr(), k_out=d["turned"].data_ptr() + at * size,
                                         q_out_stride=self.width, k_out_stride=self.width)
        self.append_io = gatgpu.AppendIO(precision=precision, rows=rows, k=d["turned"].data_ptr() + at * size, v=d["qkv"].data_ptr() + v * size,
                                         k_stride=self.width, v_stride=self.width, slot=d["slot"].data_ptr())
        self.attention_io = gatgpu.CacheAttentionIO(precision=precision, heads=heads, scale=self.scale, rows=rows, requests=requests, most=most, blocks=blocks,
                                                    table_stride=blocks, q=d["turned"].data_ptr(), q_stride=self.width, q_begin=d["q_begin"].data_ptr(),
                                                    k_len=d["k_len"].data_ptr(), table=d["table"].data_ptr(), out=d["out"].data_ptr(), out_stride=heads * dim,
                                                    lse=d["lse"].data_ptr())
        self.work = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (ctx.blocks_workspace(self.blocks_io),
                                                                                    ctx.cache_attention_workspace(d["cache"], self.attention_io))]
        torch.cuda.synchronize()

    def enqueue(self):
        self.ctx.blocks_assign(self.blocks_io, self.work[0].data_ptr(), self.work[0].numel())
        self.ctx.rotate_forward(self.rotate_io)
        self.ctx.cache_append(self.d["cache"], self.append_io)
        self.ctx.cache_attention(self.d["cache"], self.attention_io, self.work[1].data_ptr(), self.work[1].numel())

    def step(self, fresh, run):
        """`fresh` new tokens of each request, through `run`; checked stage by stage, each against the plain form of what the one before left."""
        d = self.d
        qkv = (normal(self.g, self.rows, self.width) * 1.5).to(TYPE[self.precision])
        d["qkv"].copy_(qkv)
        d["fresh"].copy_(words(fresh))
        d["out"].fill_(7)
        d["lse"].fill_(7)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        want = assign(self.cached, fresh, self.table, self.free, self.count, self.page, self.pages, self.blocks, self.rows)
        for name, at in (("stored", "cached"), ("free_left", "free_count"), ("k_len",) * 2, ("q_begin",) * 2, ("slot",) * 2, ("position",) * 2, ("unserved",) * 2):
            assert host(d[at]).tolist() == want[name], name
        assert host(d["table"]).tolist() == [x for row in self.table for x in row]
        self.cached, self.count = want["stored"], want["free_left"][0]
        h, hk, n = self.heads, self.kv_heads, self.rows
        turned = d["turned"].cpu()
        parts = [x.view(n, -1, self.dim) for x in turned[:, :(h + hk) * self.dim].split([h * self.dim, hk * self.dim], 1)]
        for got, x, gamma in zip(parts, qkv[:, :(h + hk) * self.dim].split([h * self.dim, hk * self.dim], 1), self.gamma):
            x = x.reshape(n, -1, self.dim).double()
            y = rotate(x, gamma.double(), self.eps, True, torch.tensor(want["position"]), self.freq, self.rot, self.pairs)
            assert bool(((got.double() - y).abs() <= rotate_bound(x, y, gamma.double(), self.eps, True, self.rot, self.pairs, self.precision)).all())
        self.host.append(parts[1], qkv[:, (h + hk) * self.dim:].reshape(n, hk, self.dim), torch.tensor(want["slot"]))
        self.host.same_values(d)
        begin = [min(b, n) for b in want["q_begin"]]
        check_attention(self.host, parts[0], begin, want["k_len"], self.table, self.scale, self.precision, d["out"].cpu().view(n, h, self.dim), d["lse"].cpu(), self.most)
        return want

    def end(self, which):
        """Requests end: their pages go back, and their places are free for others."""
        gone = [c if r in which else 0 for r, c in enumerate(self.cached)]
        self.d["gone"].copy_(words(gone))
        torch.cuda.synchronize()
        self.ctx.blocks_release(self.release_io, self.work[0].data_ptr(), self.work[0].numel())
        self.ctx.synchronize()
        self.count = release(gone, self.table, self.free, self.count, self.page, self.pages, self.blocks)
        assert host(self.d["free"])[:self.count].tolist() == self.free[:self.count] and host(self.d["free_count"])[0] == self.count
        for r in which:
            self.cached[r] = 0
        self.d["cached"].copy_(words(self.cached))
        torch.cuda.synchronize()

    def evict(self, r, b):
        """One block of a request is given up: hidden from then on."""
        self.table[r][b] = NONE
        self.d["table"].view(self.requests, self.blocks)[r, b] = -1
        torch.cuda.synchronize()


@pytest.mark.parametrize("precision,pairs", [(FP, HALVES), (BF, NEIGHBOURS)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("most", [8, 60, 200])
def test_steps_of_a_server(ctx, precision, pairs, page, most):
    """Prompts in parts, tokens one by one, requests that find no page, that end and that begin: one captured step, replayed."""
    pages = 24 * 16 // page
    s = Server(ctx, precision, requests=5, rows=90, most=most, page=page, pages=pages, blocks=256 // page, heads=4, kv_heads=2, dim=32, pairs=pairs, seed=page + most)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(ctx.stream())
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        s.enqueue()
    part = min(most, 40)
    s.step([part, 3, 0, 0, 1], graph.replay)
    s.step([min(part, 20), 1, part, 0, 1], graph.replay)
    s.step([0, 0, 0, 0, 0], graph.replay)
    for i in range(3):
        s.step([1, 1, 1, min(most, 9 + i), 1], graph.replay)
    s.step([1, 1, 1, 1, 1], s.enqueue)  # (eager between the replays)
    s.end([0, 3])
    s.step([min(most, 30), 1, 1, 0, 0], graph.replay)
    s.evict(2, 0)
    s.step([1, 2, 1, min(most, 17), 1], graph.replay)
    unserved = 0
    for _ in range(12 * max(1, 8 // most)):  # until pages or table rows run out
        unserved += s.step([min(most, 25), 1, min(most, 30), 1, min(most, 20)], graph.replay)["unserved"][0]
    assert unserved > 0 or most < 20
    s.end([0, 1, 2, 3, 4])
    assert s.count == pages - 1  # (all but the block that was given up)
    s.step([1, 1, 1, 1, 1], graph.replay)


@pytest.mark.parametrize("precision", [FP, BF])
def test_two_captured_servers(ctx, precision):
    """Two graphs, a workspace and a cache each, replayed in turn without waiting between."""
    both = [Server(ctx, precision, requests=3, rows=40, most=m, page=16, pages=30, blocks=20, heads=4, kv_heads=2, dim=64, pairs=HALVES, seed=m) for m in (4, 40)]
    graphs, stream = [], torch.cuda.ExternalStream(ctx.stream())
    for s in both:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            s.enqueue()
        graphs.append(graph)

    def replay_both():  # the other's step first, of no tokens
        for g in graphs:
            g.replay()

    for fresh in ([4, 1, 2], [1, 1, 1], [3, 0, 4]):
        for s, other in zip(both, both[::-1]):
            other.d["fresh"].zero_()
            torch.cuda.synchronize()
            s.step(fresh, replay_both)


@pytest.mark.parametrize("precision,pairs", [(FP, NEIGHBOURS), (BF, HALVES)])
@pytest.mark.parametrize("dim,heads,kv_heads", [(32, 4, 2), (64, 3, 3), (128, 4, 1)])
def test_training_through_attention(ctx, precision, pairs, dim, heads, kv_heads):
    """Rotation in front of attention among the rows of segments, forward and backward, on rows of queries, keys and values side by side."""
    lens = [33, 1, 70, 5]
    n = sum(lens)
    p = RotateProblem(n, heads, kv_heads, dim, precision, pairs=pairs, seed=dim)
    p.position = torch.cat([torch.arange(x, dtype=torch.int32) for x in lens])
    d = p.device()
    width, hq, hk = p.x.shape[1], heads * dim, (heads + kv_heads) * dim
    a = AttentionProblem(lens, lens, heads, kv_heads, dim, precision, mask=gatgpu.MASK_PREFIX, seed=dim)
    torch.cuda.synchronize()
    ctx.rotate_forward(p.io(d))
    ctx.synchronize()
    rows = d["y"]
    rows[:, hk:] = d["x"][:, hk:]  # values stand beside the turned queries and keys
    a.q, a.k, a.v = (x.unflatten(1, (-1, dim)) for x in (rows[:, :hq], rows[:, hq:hk], rows[:, hk:hk + kv_heads * dim]))
    out, io = a.buffers()
    io.dq, io.dk, io.dv = (d["dy"].data_ptr() + x * d["dy"].element_size() for x in (0, hq, hk))
    io.dq_stride = io.dk_stride = io.dv_stride = width
    back = p.io(d, True)
    with a.plan(ctx) as plan:
        ws = torch.empty(max(1, plan.workspace_bytes(), plan.workspace_bytes(backward=True), ctx.rotate_workspace(back)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        plan.forward(io, ws.data_ptr(), ws.numel())
        plan.backward(io, ws.data_ptr(), ws.numel())
        ctx.rotate_backward(back, ws.data_ptr(), ws.numel())
        ctx.synchronize()
    out.update(dq=d["dy"][:, :hq].unflatten(1, (-1, dim)), dk=d["dy"][:, hq:hk].unflatten(1, (-1, dim)), dv=d["dy"][:, hk:].unflatten(1, (-1, dim)))
    a.check(out)
    p.dy = d["dy"].cpu()  # what attention left for the rotation
    p.check(d, in_place=True)
    assert math.isfinite(float(d["dx"][:, :hk].float().abs().max()))
