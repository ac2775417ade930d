"""Refusals of the paged cache's operators at the edges of what they take, without a GPU (nothing is launched)."""

import ctypes as C
import math

import pytest

from speech_to_speech_amd import native
from test_paged import P, handle


def attend(kv, *, scale=1.0, H=4, o_rs=None, cu=0, B=1, T=1, max_new=1, max_kv=512, ws=0, ws_bytes=0):
    return native.load().s2s_op_attn_paged(None, C.byref(kv), P, H * 128, P, H * 128 if o_rs is None else o_rs, H, P, 8, P, cu, B, T, max_new, max_kv, scale, 1, 0, ws, ws_bytes)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38])
def test_scales_that_are_no_numbers_are_refused(scale):
    assert attend(handle(), scale=scale) == -1 and b"scale" in native.load().s2s_last_error()


def test_more_workgroups_than_a_launch_takes_are_refused():
    """A launch has fewer than 2^32 work-items along a dimension: 2^24 workgroups of 256 are too many."""
    lib, kv = native.load(), handle(kv_heads=8)
    sizes = lambda B, rows: lib.s2s_op_attn_paged_ws(C.byref(kv), 16, B, rows, rows, 512, 1, 0)  # noqa: E731
    assert sizes(2048, 2**16 - 128) == 0
    assert sizes(2048, 2**16) == -1 and b"too many" in lib.s2s_last_error()
    assert sizes(2048, 2**17) == -1 and b"too many" in lib.s2s_last_error()
    assert attend(kv, H=16, cu=P, B=2048, T=2**17, max_new=2**17) == -1 and b"too many" in lib.s2s_last_error()
    # the second launch of split calls goes over all rows and heads
    one = handle(kv_heads=1)
    assert lib.s2s_op_attn_paged_ws(C.byref(one), 64, 1, 2**19, 1, 2**20, 1, 0) > 0
    assert lib.s2s_op_attn_paged_ws(C.byref(one), 64, 1, 2**20, 1, 2**20, 1, 0) == -1 and b"too many" in lib.s2s_last_error()
