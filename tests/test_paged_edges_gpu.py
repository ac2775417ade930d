"""Attention over the paged cache at the edges of what its documentation allows: scales of any sign, sessions beyond the host's bounds, windows of any size;
against plain implementations in 64 bits (tests/paged_reference.py)."""

import ctypes as C

import pytest
import torch

import paged_reference as R
from speech_to_speech_amd import native
from speech_to_speech_amd.paged_kv import rope_tables
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


# ---- sessions beyond the host's bounds --------------------------------------------------------------------------------------------------------

CUTS = [  # new rows, bound of the new rows, positions, bound of the positions, Hkv, H, D, ps
    ([9, 1, 4], 3, [200, 64, 4], 200, 2, 4, 64, 64),              # single rows' kernel, one walk
    ([2, 3], 1, [70, 3], 70, 1, 2, 128, 64),
    ([9, 1], 3, [1500, 64], 1500, 2, 4, 64, 64),                  # a few splits
    ([9, 2], 3, [4000, 2], 4000, 1, 4, 64, 64),                   # many
    ([130, 70], 80, [200, 70], 200, 2, 4, 128, 64),               # prompts' kernel
    ([100, 3], 70, [3000, 5], 3000, 1, 2, 64, 64),                # in splits
    ([5, 1], 9, [300, 64], 230, 2, 4, 64, 64),                    # more positions than the bound
    ([9, 40], 7, [300, 100], 64, 1, 4, 64, 64),                   # both; some rows' own positions lie behind the bound
    ([150, 90], 100, [2900, 800], 2500, 1, 2, 64, 64),
    ([1, 1], 1, [900, 64], 500, 2, 4, 256, 64),
]


def attend_beyond(kind, dtype, case, causal=True, window=0, rows=None):
    """-> for every session (what the call gave for its rows, 64 bits of those within the bounds, their tolerance, its rows within the bounds)."""
    new, max_new, kv, max_kv, Hkv, H, D, ps = case
    B, cu, starts = len(new), ragged(new), ragged(kv)
    table, n_pages = make_table(kv, ps, 2, sum(kv))
    cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    k, v = randn(starts[-1], Hkv, D, seed=1, dtype=dtype), randn(starts[-1], Hkv, D, seed=2, dtype=dtype)
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32([0] * B), i32(starts), max_new=max(kv))
    kd, vd = (R.four_bit_values(x).double() for x in (k, v)) if kind == "int4" else (k.double(), v.double())
    T = cu[-1] if rows is None else rows
    q, out = randn(cu[-1], H, D, seed=3, dtype=dtype), torch.full((T + 2, H, D), 3.0, dtype=dtype, device=DEV)[:T]
    cache.attend(q[:T].to(DEV), table.to(DEV), i32(kv), i32(cu), max_new=max_new, max_kv=max_kv, causal=causal, window=window, out=out)
    got, result = out.cpu().double(), []
    for b in range(B):
        vv, r = vd[starts[b] : starts[b + 1]], slice(cu[b], cu[b + 1])
        want, size = R.attend(q[r].double(), kd[starts[b] : starts[b + 1]], vv, new[b], D**-0.5, causal, window, torch.arange(kv[b]) < max_kv)
        result.append((got[r], want, tolerance(want, size, kind, dtype, float(vv.abs().max()), kv[b], D, False), min(new[b], max_new, T - cu[b])))
    return result


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("case", CUTS)
def test_rows_within_the_bounds_see_what_they_see_without_bounds(kind, dtype, case):
    """A session with more new rows or positions than the host's bounds: the rows that are computed keep their place in the session."""
    for mask in (dict(), dict(window=40), dict(causal=False)):
        for b, (got, want, tol, n) in enumerate(attend_beyond(kind, dtype, case, **mask)):
            assert ((got[:n] - want[:n]).abs() <= tol[:n]).all(), (mask, b)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_rows_of_a_session_that_ends_behind_the_row_buffer_keep_their_place(kind, dtype):
    for case, rows in ((([5, 9], 9, [300, 90], 300, 2, 4, 64, 64), 11), (([50, 90], 90, [300, 190], 300, 2, 4, 64, 64), 130)):
        for got, want, tol, n in attend_beyond(kind, dtype, case, rows=rows):
            assert ((got[:n] - want[:n]).abs() <= tol[:n]).all()


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("case", CUTS)
def test_rows_beyond_the_bound_are_left_as_they_are(kind, dtype, case):
    for mask in (dict(), dict(window=40), dict(causal=False)):
        for b, (got, _, _, n) in enumerate(attend_beyond(kind, dtype, case, **mask)):
            assert (got[n:] == 3).all(), (mask, b)


# ---- the C entry points -------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("new,kv", [(9, 3), (130, 100), (1, 64)])
def test_a_window_of_the_largest_integer_hides_nothing(new, kv):
    """Also for rows in front of the first position."""
    Hkv, H, D = 1, 2, 64
    table, n_pages = make_table([kv], 64, 0, 1)
    tb = table.to(DEV)
    cache = poisoned(n_pages, Hkv, D, 64, "model", F32)
    cache.append(randn(kv, Hkv, D, seed=1).to(DEV), randn(kv, Hkv, D, seed=2).to(DEV), tb, i32([0]), i32([0, kv]), max_new=kv)
    q, lens, cu = randn(new, H, D, seed=3).to(DEV), i32([kv]), i32([0, new])
    outs = []
    for window in (1 << 29, 2**31 - 1):
        out = torch.full_like(q, 3.0)
        st = native.load().s2s_op_attn_paged(torch.cuda.current_stream().cuda_stream, C.byref(cache._kv), q.data_ptr(), H * D, out.data_ptr(), H * D, H, tb.data_ptr(), tb.shape[1],
                                             lens.data_ptr(), cu.data_ptr(), 1, new, new, kv, 0.125, 1, window, 0, 0)
        assert st == 0, native.load().s2s_last_error()
        outs.append(out)
    assert torch.equal(*outs) and float(outs[0][-1].abs().max()) > 0


def test_an_append_without_queries_takes_any_stride_of_theirs():
    cache, other = (poisoned(2, 1, 64, 64, "model", F32) for _ in range(2))
    k, v, table, start = randn(2, 1, 64, seed=1).to(DEV), randn(2, 1, 64, seed=2).to(DEV), i32([[0], [1]]), i32([3, 5])
    cache.append(k, v, table, start)
    st = native.load().s2s_op_kv_append_paged(torch.cuda.current_stream().cuda_stream, C.byref(other._kv), k.data_ptr(), 64, v.data_ptr(), 64, 0, 7, 0, 64, 0, table.data_ptr(), 1,
                                              start.data_ptr(), 0, 2, 2, 1, 0, 0, 0, 0, 0)
    assert st == 0, native.load().s2s_last_error()
    assert torch.equal(cache.k.view(torch.uint8), other.k.view(torch.uint8)) and torch.equal(cache.v.view(torch.uint8), other.v.view(torch.uint8))


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_a_bound_of_no_new_rows_leaves_everything_as_it_is(kind, dtype):
    cache = poisoned(4, 2, 64, 64, kind, dtype)
    before = [t.clone() for t in (cache.k, cache.v)]
    rows, table, start, cu = randn(3, 2, 64, seed=1, dtype=dtype).to(DEV), i32([[0, 1], [2, 3]]), i32([3, 64]), i32([0, 1, 3])
    cos, sin = rope_tables(64, 128, device=DEV)
    out = torch.full_like(rows, 7.0)
    assert cache.append(rows, rows, table, start, cu, max_new=0, cos=cos, sin=sin, q=rows, q_out=out) is out
    assert cache.attend(rows, table, start, cu, max_new=0, out=out) is out
    assert all(x.shape == rows.shape for x in cache.read(table, start, cu, 3, max_new=0))
    assert (out == 7).all() and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (cache.k, cache.v)))
