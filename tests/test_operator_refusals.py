"""Entries of attention and layer norm without a context or a plan: refused, with a message, without a GPU."""
import ctypes

import pytest

import gatgpu


@pytest.mark.parametrize("name,args", [
    ("gatgpu_attention_create", (None, None, 0, None, None, None, None, None, None)),
    ("gatgpu_attention_workspace", (None, None, None)),
    ("gatgpu_attention_distances", (None, None, None, None)),
    ("gatgpu_attention_forward", (None, None, None, 0)),
    ("gatgpu_attention_backward", (None, None, None, 0)),
    ("gatgpu_norm_forward", (None, None)),
    ("gatgpu_norm_backward", (None, None, None, 0)),
    ("gatgpu_norm_workspace", (None, 1, 1, None)),
    ("gatgpu_set_norm", (None, 0, None, None, 0.0)),
])
def test_null_handles(name, args):
    lib = gatgpu.load_library()
    assert getattr(lib, name)(*args) == gatgpu.EINVAL
    assert b"null" in lib.gatgpu_last_error(None)


def test_destroying_no_plan_is_fine():
    assert gatgpu.load_library().gatgpu_attention_destroy(None) == gatgpu.OK


def test_a_plan_outlives_neither_its_context_nor_itself():
    class Closed:
        h, _check = None, None

    plan = object.__new__(gatgpu.Attention)
    plan.ctx, plan.lib, plan.segments = Closed(), gatgpu.load_library(), 0
    for handle in (None, ctypes.c_void_p(16)):
        plan.h = handle
        for call in (plan.workspace_bytes, plan.distance_layout, lambda: plan.forward(None), lambda: plan.backward(None)):
            with pytest.raises(ValueError):
                call()
    plan.close()  # (its context is gone: nothing to free on it)
    assert plan.h is None
