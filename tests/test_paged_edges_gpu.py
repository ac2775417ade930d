"""Attention over the paged cache at the edges of what its documentation allows: scales of any sign, sessions beyond the host's bounds, windows of any size;
against plain implementations in 64 bits (tests/paged_reference.py)."""

import ctypes as C

import pytest
import torch

import paged_reference as R
from speech_to_speech_amd import native
from test_paged_gpu import BF, DEV, F32, KINDS, check_attention, i32, make_table, poisoned, ragged, randn, tolerance

pytestmark = pytest.mark.gpu


# ---- scales ---------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.125, -1.5, 1e-40, -1e-40])
def test_attend_with_any_finite_scale(kind, dtype, scale):
    """Zero weighs every position that is seen alike, a negative scale prefers the smallest product; hidden positions stay hidden."""
    check_attention([1] * 4, [203, 64, 1, 0], 2, 4, 64, 64, kind, dtype, scale=scale)
    check_attention([1, 1], [5000, 17], 1, 20, 64, 256, kind, dtype, scale=scale, window=3000, seed=1)
    check_attention([1, 1], [700, 64], 2, 14, 256, 64, kind, dtype, scale=scale, causal=False, seed=2, aligned=False, max_kv=704)
    check_attention([40, 0, 65], [40, 9, 300], 2, 4, 128, 64, kind, dtype, scale=scale, few=False, seed=3)
    check_attention([130, 7], [129, 3], 2, 2, 64, 64, kind, dtype, scale=scale, few=False, window=50, seed=4, aligned=False)
    check_attention([40], [4100], 1, 2, 64, 64, kind, dtype, scale=scale, few=False, seed=5)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("size,scale", [(2.0**-100, 1e-12), (2.0**-120, 1e-20), (2.0**-126, -1e-38)])
def test_attend_4_bits_with_queries_near_the_smallest_float(rows, size, scale):
    """Scores of nothing but zeros in 32 bits: every seen position weighs the same, whatever their scale comes to."""
    Hkv, D, ps, n = 2, 64, 64, 150
    table, n_pages = make_table([n], ps, 0, 1)
    cache = poisoned(n_pages, Hkv, D, ps, "int4")
    k, v = randn(n, Hkv, D, seed=1, dtype=BF), randn(n, Hkv, D, seed=2, dtype=BF)
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32([0]), i32([0, n]), max_new=n)
    q = (randn(rows, 4, D, seed=3).clamp(-2, 2) * size).to(BF)
    o = cache.attend(q.to(DEV), table.to(DEV), i32([n]), i32([0, rows]), max_new=rows, scale=scale).cpu().double()
    kd, vd = R.four_bit_values(k).double(), R.four_bit_values(v).double()
    want, weight = R.attend(q.double(), kd, vd, rows, scale)
    assert ((o - want).abs() <= tolerance(want, weight, "int4", BF, float(vd.abs().max()), n, D, False)).all()
