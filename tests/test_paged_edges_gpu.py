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


# ---- what looser tolerances would let pass --------------------------------------------------------------------------------------------------------


def exact_rows(n, Hkv, D, seed, step):
    """Rows whose every 4-bit group holds (code - 8) step exactly: codes 0 and 15 are in it, so its scale is the power of two `step` and its zero 0."""
    c = torch.randint(0, 16, (n, Hkv, D), generator=torch.Generator().manual_seed(seed)).double()
    c[..., ::32], c[..., 1::32] = 0, 15
    return (c - 8) * step


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,kv,Hkv,H,D,few", [([1, 1], [333, 64], 1, 2, 128, True), ([1], [2100], 2, 4, 64, True), ([40, 130], [200, 333], 1, 2, 128, False),
                                               ([70], [2500], 1, 1, 64, False)])
def test_attend_with_a_rising_maximum_of_exact_scores(kind, dtype, new, kv, Hkv, H, D, few):
    """Products that every type holds exactly and that grow along the session to thousands, so that the running maximum is raised again and again.  What is left are the
    roundings of the scaling: the factor of the scores (2 half steps of it), the scaled maximum, its bias and the argument of exp2 (one each) of at most the largest
    |score|, so 8 half steps of f32 of that with room; weights as in `tolerance`."""
    B, cu, starts, ps = len(new), ragged(new), ragged(kv), 64
    table, n_pages = make_table(kv, ps, 2, 1)
    cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    k = torch.cat([exact_rows(n, Hkv, D, 1 + b, 1.0) * 2.0 ** torch.div(torch.arange(n) * 8, n, rounding_mode="floor")[:, None, None] for b, n in enumerate(kv)])
    v = exact_rows(starts[-1], Hkv, D, 7, 0.125)
    q = torch.randint(-8, 9, (cu[-1], H, D), generator=torch.Generator().manual_seed(5)).double() / 4
    assert torch.equal(R.four_bit_values(k.to(BF)).double(), k) and torch.equal(R.four_bit_values(v.to(BF)).double(), v)
    cache.append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), table.to(DEV), i32([0] * B), i32(starts), max_new=max(kv))
    for scale in (1.0, -0.5, 0.01):
        o = cache.attend(q.to(dtype).to(DEV), table.to(DEV), i32(kv), i32(cu), max_new=max(new), max_kv=max(kv), scale=scale).cpu().double()
        for b in range(B):
            qq, kk, vv = q[cu[b] : cu[b + 1]], k[starts[b] : starts[b + 1]], v[starts[b] : starts[b + 1]]
            want, _ = R.attend(qq, kk, vv, new[b], scale)
            top = max(float((qq[:, h] @ kk[:, h * Hkv // H].T).abs().max()) for h in range(H)) * abs(scale)
            zero = torch.zeros(new[b], H, dtype=torch.float64)
            tol = tolerance(want, zero, kind, dtype, 1.0, kv[b], D, few) + 2 * 8 * 2.0**-24 * top
            assert float(tol.max()) < 0.05 and float(want.abs().max()) > 0.3 and top > 3000 * abs(scale)     # a wrong row or none at all is far outside
            assert ((o[cu[b] : cu[b + 1]] - want).abs() <= tol).all(), (scale, b, float(((o[cu[b] : cu[b + 1]] - want).abs() / tol).max()))


@pytest.mark.parametrize("rows,new,B,Hkv", [(16, 1, 64, 1), (17, 1, 63, 1), (24, 1, 2, 1), (33, 1, 2, 1), (64, 1, 2, 1), (40, 20, 3, 2), (64, 64, 5, 1), (20, 1, 7, 9)])
def test_single_rows_kernel_keeps_what_the_first_rounding_of_a_weight_leaves(rows, new, B, Hkv):
    """bf16, up to 64 (row, head) pairs per KV head and fewer than 64 (session, KV head) pairs (up to 16: any number): a weight is two operands.  Values of one sign and
    the other whose weights nearly cancel, so that a weight rounded once would show."""
    assert rows <= 16 or (rows <= 64 and B * Hkv < 64)
    G, D, ps, n = rows // new, 64, 64, 96
    kv = [n] * B
    table, n_pages = make_table(kv, ps, 0, rows)
    cache = poisoned(n_pages, Hkv, D, ps, "model", BF)
    half = randn(B * n // 2, Hkv, D, seed=1)
    k = torch.stack([half, half + 0.02 * randn(*half.shape, seed=2)], 1).flatten(0, 1).to(BF)
    sign = torch.randint(0, 2, half.shape, generator=torch.Generator().manual_seed(3)).float() * 2 - 1
    v = torch.stack([sign, -sign], 1).flatten(0, 1).to(BF)
    q = randn(B * new, Hkv * G, D, seed=4, dtype=BF, scale=0.2)
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32([0] * B), i32(ragged(kv)), max_new=n)
    o = cache.attend(q.to(DEV), table.to(DEV), i32(kv), i32(ragged([new] * B)), max_new=new, max_kv=n, causal=False).cpu().double()
    for b in range(B):
        qq, kk, vv = q[b * new : (b + 1) * new].double(), k[b * n : (b + 1) * n].double(), v[b * n : (b + 1) * n].double()
        want, size = R.attend(qq, kk, vv, new, D**-0.5, causal=False)
        tol = tolerance(want, size, "model", BF, 1.0, n, D, True)
        assert ((o[b * new : (b + 1) * new] - want).abs() <= tol).all(), b
        if b == 0:      # the same in 64 bits with weights rounded once to bf16 is outside
            p = torch.exp(qq[:, 0] @ kk[:, 0].T * D**-0.5)
            once = (p / p.amax(-1, keepdim=True)).to(BF).double()
            off = (once @ vv[:, 0] / (p / p.amax(-1, keepdim=True)).sum(-1, keepdim=True) - want[:, 0]).abs()
            assert (off > tol[:, 0]).any()


# ---- what stands together in one call -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_single_rows_beside_a_prompt(kind, dtype):
    """The usual batch of a serving loop: a prompt joins sessions that are taking single steps."""
    kv = [1 + 37 * i % 700 for i in range(47)]
    check_attention([1] * 23 + [300] + [1] * 24, kv[:23] + [410] + kv[23:], 2, 4, 64, 64, kind, dtype, few=False)
    check_attention([1] * 8 + [70, 130], kv[:8] + [1500, 130], 1, 2, 128, 64, kind, dtype, few=False, seed=3)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,kv,at", [(1, 70, 5), (70, 70, 30), (3, 2100, 2098), (90, 2600, 2550), (90, 2600, 100)])
def test_an_infinite_score_is_nan_where_it_is_seen_and_nothing_elsewhere(kind, dtype, new, kv, at):
    """exp(inf - inf) is NaN for the rows that see the key (a 4-bit group with an infinity holds NaN).  Rows before it stay within the tolerance of the call without it: a
    wave raises the running maxima of its 16 or 32 columns together, at other tiles then, so each weight is a multiple of another 2^-m before it is rounded and
    what `tolerance` counts is the same.  Another session is bit for bit what it was."""
    Hkv, H, D, ps = 1, 2, 64, 64
    table, n_pages = make_table([kv, kv], ps, 0, kv)
    cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    k, v = randn(2 * kv, Hkv, D, seed=1, dtype=dtype), randn(2 * kv, Hkv, D, seed=2, dtype=dtype)
    q = randn(2 * new, H, D, seed=3, dtype=dtype)
    q[..., 7] = 1.0
    plain = k.clone()
    k[at, 0, 7] = float("inf")
    outs = []
    for rows in (plain, k):
        cache.append(rows.to(DEV), v.to(DEV), table.to(DEV), i32([0, 0]), i32([0, kv, 2 * kv]), max_new=kv)
        outs.append(cache.attend(q.to(DEV), table.to(DEV), i32([kv, kv]), i32([0, new, 2 * new]), max_new=new, max_kv=kv).cpu())
    blind = max(0, at - (kv - new))      # rows of the first session that do not see the key
    assert torch.isnan(outs[1][blind:new]).all() and torch.isfinite(outs[0]).all()
    assert torch.equal(outs[1][new:], outs[0][new:])
    kd, vd = (R.four_bit_values(x[:kv]).double() for x in (plain, v)) if kind == "int4" else (plain[:kv].double(), v[:kv].double())
    want, size = R.attend(q[:new].double(), kd, vd, new, D**-0.5)
    tol = tolerance(want, size, kind, dtype, float(vd.abs().max()), kv, D, False)
    for o in outs:
        n = new if o is outs[0] else blind
        assert ((o[:n].double() - want[:n]).abs() <= tol[:n]).all()


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [203, 64, 0]), ([1, 1], [4000, 3]), ([40, 0, 65], [40, 9, 300]), ([130, 7], [129, 3]), ([90], [3000])])
def test_results_in_place_of_their_queries(kind, dtype, new, kv):
    Hkv, H, D, B = 2, 4, 128, len(new)
    table, n_pages = make_table(kv, 64, 0, 1)
    cache, tb, lens, cu = poisoned(n_pages, Hkv, D, 64, kind, dtype), table.to(DEV), i32(kv), i32(ragged(new))
    cache.append(randn(sum(kv), Hkv, D, seed=1, dtype=dtype).to(DEV), randn(sum(kv), Hkv, D, seed=2, dtype=dtype).to(DEV), tb, i32([0] * B), i32(ragged(kv)), max_new=max(kv))
    q = randn(sum(new), H, D, seed=3, dtype=dtype).to(DEV)
    want = cache.attend(q, tb, lens, cu, max_new=max(new), max_kv=max(kv))
    assert cache.attend(q, tb, lens, cu, max_new=max(new), max_kv=max(kv), out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_a_captured_prompt_replays_beyond_its_bounds(kind, dtype):
    """Lengths on the device pass the bounds of the capture and come back: every replay against the eager call, rows beyond left alone."""
    Hkv, H, D, kvs = 2, 4, 64, [700, 3000]
    table, n_pages = make_table(kvs, 64, 0, 1)
    cache, tb = poisoned(n_pages, Hkv, D, 64, kind, dtype), table.to(DEV)
    cache.append(randn(sum(kvs), Hkv, D, seed=1, dtype=dtype).to(DEV), randn(sum(kvs), Hkv, D, seed=2, dtype=dtype).to(DEV), tb, i32([0, 0]), i32(ragged(kvs)), max_new=max(kvs))
    q, lens, cu = torch.zeros(200, H, D, dtype=dtype, device=DEV), i32([600, 2500]), i32([0, 50, 130])
    args, out = dict(max_new=80, max_kv=2600), torch.zeros_like(q)
    ws = torch.zeros(max(16, cache.workspace_bytes(H, 2, 200, **args)), dtype=torch.uint8, device=DEV)
    cache.attend(q, tb, lens, cu, out=out, workspace=ws, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        cache.attend(q, tb, lens, cu, out=out, workspace=ws, **args)
    for i, (kv, new) in enumerate((([600, 2500], [50, 80]), ([700, 3000], [120, 80]), ([700, 2600], [20, 170]), ([90, 2601], [80, 81]), ([600, 2500], [50, 80]))):
        q.copy_(randn(200, H, D, seed=10 + i, dtype=dtype))
        lens.copy_(i32(kv))
        cu.copy_(i32(ragged(new)))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(out, 3.0)
        cache.attend(q, tb, lens, cu, out=want, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        at = 0
        for n in new:
            assert (out[at : at + min(n, 80)] != 3).any(-1).all() and (out[at + min(n, 80) : at + n] == 3).all()
            at += n
        assert (out[at:] == 3).all()
