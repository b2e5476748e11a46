"""Block tables of more requests than are summed at a time (4096): the list of free pages goes on from one pass to the next."""
import numpy as np
import pytest
import torch

import gatgpu
from test_gpu_blocks import Problem, back

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def held_once(p, d, left):
    """No page stands twice among the tables' blocks that hold tokens and the list."""
    table, stored = back(d["table"])[:len(p.cached) * p.stride].reshape(len(p.cached), p.stride), back(d["stored"])[:len(p.cached)]
    used = [table[r, :-(-int(n) // p.page)] for r, n in enumerate(stored)]
    pages = np.concatenate(used + [back(d["free"])[:left]])
    assert pages.max() < p.pages and np.unique(pages).size == pages.size


def two_steps(ctx, p, fresh):
    """A step, and another on the lengths, the table and the list that it leaves."""
    d = p.run(ctx)
    want = p.check(d)
    left = want["free_left"][0]
    held_once(p, d, left)
    p.table = back(d["table"])[:len(p.cached) * p.stride].reshape(len(p.cached), p.stride).tolist()
    p.cached, p.fresh, p.count, p.rows = want["stored"], list(fresh), left, sum(fresh) + 3
    d = p.run(ctx)
    held_once(p, d, p.check(d)["free_left"][0])
    return want


@pytest.mark.parametrize("requests", [4095, 4096, 4097, 4100, 5000, 8193, 20_000])
def test_every_request_takes_a_page(ctx, requests):
    p = Problem([0] * requests, [1] * requests, spare=2 * requests + 2, blocks=2, seed=requests)
    assert two_steps(ctx, p, [16] * requests)["free_left"] == [requests + 2]


@pytest.mark.parametrize("requests,first,last", [(4097, 0, 0), (4097, 4095, 4096), (5000, 4000, 4100), (9000, 4090, 8195), (9000, 8191, 8192), (20_000, 12_288, 12_300)])
def test_some_requests_take_pages(ctx, requests, first, last):
    """The last one that does stands in another pass, or in another lane, than the requests before it."""
    fresh = [1 if first <= r <= last else 0 for r in range(requests)]
    p = Problem([0] * requests, fresh, spare=requests + 20, blocks=2, seed=requests + last)
    two_steps(ctx, p, [1 if r % 3 else 0 for r in range(requests)])


@pytest.mark.parametrize("requests,spare", [(5000, 4096), (5000, 4099), (9000, 4500), (9000, 8192), (9000, 100), (20_000, 19_999)])
def test_pages_run_short_in_a_later_pass(ctx, requests, spare):
    p = Problem([0] * requests, [1] * requests, spare=spare, blocks=2, seed=spare)
    want = two_steps(ctx, p, [16] * requests)
    assert want["free_left"] == [0] and want["unserved"] == [requests - spare]


def test_lengths_of_all_kinds(ctx):
    rng = np.random.default_rng(7)
    for requests in (4500, 13_000):
        cached, fresh = rng.integers(0, 60, requests).tolist(), (rng.integers(0, 40, requests) * rng.integers(0, 2, requests)).tolist()
        need = sum(-(-(c + f) // 16) + (-c // 16) for c, f in zip(cached, fresh))
        for spare in (need + requests, need // 2):
            p = Problem(cached, fresh, spare=spare, blocks=9, seed=requests)
            two_steps(ctx, p, rng.integers(0, 20, requests).tolist())
