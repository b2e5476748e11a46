"""Cached attention where the scales of the pages that a row sees are far apart: in each of its forms, against the plain form in 64 bits."""
import math

import pytest
import torch

import gatgpu
from cache_cases import EPS, Serving, generator, values

pytestmark = pytest.mark.gpu

BF, FP = gatgpu.BF16, gatgpu.FP32
NONE = gatgpu.NO_PAGE
FORMS = [(FP, 16), (FP, 40), (FP, 400), (BF, 16), (BF, 40), (BF, 400)]
forms = pytest.mark.parametrize("precision,most", FORMS)
# Tokens and rows of requests: tables that a block takes alone, and work that is cut between blocks and joined.
SHORT, LONG = ([400, 77, 0], [16, 3, 0]), ([9000, 5000, 33], [16, 9, 2])


@pytest.fixture(scope="module")
def ctx():
    c = gatgpu.Context(0)
    yield c
    c.close()


def blocks_of(p, r):
    return [b for b in p.table[r] if b != NONE]


def small_first(pages, g):
    return [-64 if i < len(pages) // 2 else 64 for i in range(len(pages))]


def large_first(pages, g):
    return [64 if i < len(pages) // 2 else -64 for i in range(len(pages))]


def one_large_last(pages, g):
    return [64 if i == len(pages) - 1 else -64 for i in range(len(pages))]


def one_large_first(pages, g):
    return [64 if i == 0 else -64 for i in range(len(pages))]


def any_of_both(pages, g):
    return [64 if x else -64 for x in torch.randint(0, 2, (len(pages),), generator=g).tolist()]


def any_at_all(pages, g):
    return torch.randint(-64, 65, (len(pages),), generator=g).tolist()


def a_little_apart(pages, g):
    return torch.randint(-12, 13, (len(pages),), generator=g).tolist()


@forms
@pytest.mark.parametrize("shape", [SHORT, LONG], ids=["short", "long"])
@pytest.mark.parametrize("place", [small_first, large_first, one_large_last, one_large_first, any_of_both, any_at_all, a_little_apart])
def test_small_and_large_pages_in_one_row(ctx, precision, most, shape, place):
    """Every token counts in the weights' sum, whatever its page's scale."""
    p = Serving(*shape, 4, 2, 32, 16, precision, seed=80)
    g = generator(81)
    for r in range(len(p.k_len)):
        pages = blocks_of(p, r)
        for b, e in zip(pages, place(pages, g)):
            p.host.v_scale[b] = 2.0 ** e
    p.check(p.run(ctx, most=most))


@forms
@pytest.mark.parametrize("score", [-6.0, -14.0, -60.0])
def test_many_small_weights_on_small_pages(ctx, precision, most, score):
    """16 tokens of score 0 on a page of scale 2^64, before, between or behind thousands of a lower score on pages of 2^-64."""
    for at in (0, 200, 561):
        p = Serving([8990], [2], 2, 1, 16, 16, precision, seed=82)
        p.host.k.zero_()
        p.host.k_scale[:] = 1.0
        p.host.v_scale[:] = 2.0 ** -64
        p.host.k[:, :, :, 0] = 0x38  # 1
        p.q.zero_()
        p.q[:, :, 0] = score
        p.scale = math.log(2.0)
        large = p.table[0][at]
        p.host.k[large, :, :, 0] = 0
        p.host.v_scale[large] = 2.0 ** 64
        p.check(p.run(ctx, most=most))


@forms
@pytest.mark.parametrize("shape", [SHORT, LONG], ids=["short", "long"])
@pytest.mark.parametrize("large", [10, 30, 64])
def test_columns_that_are_zero_in_large_pages(ctx, precision, most, shape, large):
    """A column whose values in the pages of the largest scale are 0 keeps the digits of the others'."""
    p = Serving(*shape, 4, 2, 32, 16, precision, seed=83)
    for r in range(len(p.k_len)):
        for i, b in enumerate(blocks_of(p, r)):
            p.host.v_scale[b] = 1.0
            if i % 9 == 2:
                p.host.v_scale[b] = 2.0 ** large
                p.host.v[b, :, 1:] = 0
    p.check(p.run(ctx, most=most))


@forms
def test_pages_of_zeros(ctx, precision, most):
    """What append writes of values that are all 0: the least scale, beside ordinary pages and lower weights."""
    p = Serving(*LONG, 4, 2, 32, 16, precision, seed=84, size=4.0)
    for r in range(len(p.k_len)):
        for i, b in enumerate(blocks_of(p, r)):
            if i % 4:
                p.host.v_scale[b] = 2.0 ** -64
                p.host.v[b] = 0
    p.check(p.run(ctx, most=most))


@forms
def test_hidden_pages_and_nan_beside_them(ctx, precision, most):
    """Pages that nobody sees, rows that see nothing, and a NaN on a small page that some rows see."""
    p = Serving([300, 200, 40], [16, 16, 7], 4, 2, 32, 16, precision, seed=85)
    for r in range(3):
        for i, b in enumerate(blocks_of(p, r)):
            p.host.v_scale[b] = 2.0 ** (64 if i % 2 else -64)
    hidden = p.table[0][5]
    p.host.k[hidden], p.host.v[hidden] = 0x7f, 0xff
    p.table[0][5] = NONE
    p.host.v[p.table[1][190 // 16], 1, 3, 190 % 16] = 0x7f
    p.table[2] = [NONE] * len(p.table[2])
    p.check(p.run(ctx, most=most))


@forms
@pytest.mark.parametrize("size", [1e7, 1e9, 1e20])
def test_far_scores_on_pages_of_all_scales(ctx, precision, most, size):
    """Rows whose largest score is far, of one token: its value, whatever the scales of the others' pages; and finite rows beside them."""
    p = Serving([400, 90], [16, 16], 4, 2, 32, 16, precision, seed=86)
    p.host.k.zero_()
    p.host.k_scale[:] = 1.0
    for r in range(2):
        for i, b in enumerate(blocks_of(p, r)):
            p.host.v_scale[b] = 2.0 ** (64 if i % 3 else -64)
    hot = {(0, 3): 17, (0, 9): 250, (1, 12): 31}  # request, row: the token of its largest score
    p.q[:, :, 0] = 0
    for (r, i), token in hot.items():
        p.host.k[p.table[r][token // 16], :, token % 16, i + 1] = 0x38
        p.q[16 * r + i] = 0
        p.q[16 * r + i, :, i + 1] = size
    d = p.run(ctx, most=most)
    p.check(d)
    out = d["out"].cpu()[:, :128].view(32, 4, 32).double()
    assert bool(torch.isfinite(out).all())
    v, scale = p.host.sides()[1]
    for (r, i), token in hot.items():
        b = p.table[r][token // 16]
        for h in range(4):
            want = values(v[b, h // 2, token % 16]) * float(scale[b, h // 2])
            # (one weight of 2^7 to 2^15, in fp16 to 2^-11 or 2^-22, over the sum of one)
            assert bool(((out[16 * r + i, h] - want).abs() <= want.abs() * (EPS[precision] + 2.0 ** -20 + (2.0 ** -11 if precision == BF else 0))).all())
