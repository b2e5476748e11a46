"""Lengths, begins and prefixes of an attention plan: whole numbers of their type's range, as given or refused. No GPU."""
import ctypes

import numpy as np
import pytest

import gatgpu


class Recorder:
    """A context whose library keeps what a plan was asked for."""

    def __init__(self):
        self.lib, self.h, self.made = self, None, None

    def _check(self, rc):
        assert rc == 0

    def gatgpu_attention_create(self, ctx, shape, n, q_begin, q_len, k_begin, k_len, prefix, out):
        read = lambda p, t: None if p is None else list((t * n).from_address(p)) if n else []  # noqa: E731
        u32, u64 = ctypes.c_uint32, ctypes.c_uint64
        self.made = read(q_begin, u64), read(q_len, u32), read(k_begin, u64), read(k_len, u32), read(prefix, u32)
        return 0


def plan(**change):
    a = dict(q_len=[3, 4], k_len=[5, 6], heads=2, dim=8, mask=gatgpu.MASK_PREFIX)
    a.update(change)
    ctx = Recorder()
    gatgpu.Attention(ctx, a.pop("q_len"), a.pop("k_len"), **a)
    return ctx.made


def test_arguments_as_given():
    want = [0, 3], [3, 4], [0, 5], [5, 6], None
    assert plan() == want
    for t in (np.int32, np.int64, np.uint32, np.uint64, np.float64, object):
        assert plan(q_len=np.array([3, 4], t), k_len=np.array([5, 6], t)) == want
    assert plan(prefix=np.array([2, 2 ** 32 - 1]), q_begin=np.array([1, 2 ** 40])) == ([1, 2 ** 40], [3, 4], [0, 5], [5, 6], [2, 2 ** 32 - 1])
    assert plan(q_len=[], k_len=[]) == ([], [], [], [], None)
    # begins of long segments do not wrap
    assert plan(q_len=[2 ** 32 - 1] * 2)[0] == [0, 2 ** 32 - 1]


@pytest.mark.parametrize("name", ["q_len", "k_len", "prefix", "q_begin", "k_begin"])
@pytest.mark.parametrize("values", [[-1, 4], [3, 2.5], [3, float("nan")], [3, float("inf")], [3, 2 ** 64], ["3", "4"], [3 + 1j, 4]])
@pytest.mark.parametrize("array", [True, False])
def test_what_no_segment_has(name, values, array):
    with pytest.raises(ValueError):
        plan(**{name: np.array(values) if array else values})


@pytest.mark.parametrize("name", ["q_len", "k_len", "prefix"])
@pytest.mark.parametrize("value", [2 ** 32, 2 ** 32 + 4, 2 ** 63])
def test_lengths_beyond_32_bits(name, value):
    with pytest.raises(ValueError):
        plan(**{name: np.array([3, value], np.uint64)})


def test_counts_of_segments_agree():
    for change in (dict(q_len=[3]), dict(prefix=[1]), dict(k_begin=[0]), dict(q_len=[[3, 4]], k_len=[[5, 6]])):
        with pytest.raises(ValueError):
            plan(**change)
