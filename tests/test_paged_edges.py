"""Refusals of the paged cache's operators at the edges of what they take, without a GPU (nothing is launched)."""

import ctypes as C
import math

import pytest
import torch

from speech_to_speech_amd import native
from speech_to_speech_amd.paged_kv import PagedKVCache
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


def test_outputs_whose_rows_share_memory_are_refused():
    """Two rows (or heads) written to one place would leave whichever came last."""
    lib, kv, ref = native.load(), handle(), lambda: native.load().s2s_last_error()
    rope = lambda o_rs, o_hs, rows=3, heads=2: lib.s2s_op_rope(None, P, 128, 64, 2 * P, o_rs, o_hs, P, P, P, 5, rows, heads, 64, 64, 0, 0)  # noqa: E731
    for o_rs, o_hs in ((0, 64), (127, 64), (128, 0), (128, 63), (64, 191), (63, 192), (-64, 64)):
        assert rope(o_rs, o_hs) == -1 and b"share" in ref(), (o_rs, o_hs)
    for o_rs, o_hs, rows, heads in ((0, 0, 2, 1), (63, 0, 2, 1), (0, 63, 1, 2)):
        assert rope(o_rs, o_hs, rows, heads) == -1 and b"share" in ref(), (o_rs, o_hs, rows, heads)
    assert lib.s2s_op_rope(None, P, 0, 64, P, 0, 64, P, P, P, 5, 3, 2, 64, 64, 0, 0) == -1 and b"share" in ref()      # a broadcast row turned in place
    for o_rs in (0, 511, -512):
        assert attend(kv, cu=P, T=2, max_new=2, o_rs=o_rs) == -1 and b"share" in ref()
    for o_rs in (0, 255, -256):
        assert lib.s2s_op_kv_read_paged(None, C.byref(kv), P, 8, P, P, 1, 2, 2, P, P, o_rs) == -1 and b"share" in ref()
        assert lib.s2s_op_kv_append_paged(None, C.byref(kv), P, 256, P, 256, P, 256, 2 * P, o_rs, 2, P, 8, P, P, 1, 2, 2, P, P, 5, 128, 0) == -1 and b"share" in ref()


def test_negative_bounds_are_refused():
    cache = PagedKVCache(4, 2, 64, device="cpu")
    table, lens, cu, rows = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.append(rows, rows, table, lens, cu, max_new=-1), lambda: cache.read(table, lens, cu, 2, max_new=-1), lambda: cache.attend(rows, table, lens, cu, max_new=-1)):
        with pytest.raises(ValueError, match="max_new"):
            call()
