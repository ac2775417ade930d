"""Rotary positions, the paged key / value cache and the attention over it, against plain implementations in 64 bits (tests/paged_reference.py)."""

import random

import pytest
import torch

import paged_reference as R
from speech_to_speech_amd import native, paged_kv
from speech_to_speech_amd.paged_kv import PagedKVCache, rope, rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def randn(*shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def poisoned(n_pages, Hkv, D, ps, kind, dtype=BF):
    """A cache whose every byte is 0xff: NaN wherever a kernel reads what nobody wrote."""
    c = PagedKVCache(n_pages, Hkv, D, page_size=ps, kind=kind, dtype=dtype, device=DEV)
    for t in (c.k, c.v, c.k_meta, c.v_meta):
        if t is not None:
            t.view(torch.uint8).fill_(255)
    return c


def make_table(lens, ps, n_extra, seed, cols=None):
    """Pages in no order -> (table int32 [B][cols] on the host, pages in the pool)."""
    need = [-(-max(x, 0) // ps) for x in lens]
    ids = list(range(sum(need) + n_extra))
    random.Random(seed).shuffle(ids)
    cols = cols or max(need + [1])
    t = torch.full((len(lens), cols), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            t[b, j] = ids.pop()
    return t, sum(need) + n_extra


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def ragged(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


# ---- rotation -----------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,heads,D,rot,inter", [(1, 1, 64, 64, False), (3, 5, 128, 128, True), (67, 16, 128, 32, False), (130, 3, 256, 64, True), (9, 2, 80, 48, False),
                                                    (5, 3, 64, 10, False), (5, 3, 30, 30, True), (1500, 20, 128, 128, False), (2100, 20, 64, 32, True), (4, 1, 2, 2, False)])
def test_rope_equals_plain_float32_and_is_near_64_bits(dtype, rows, heads, D, rot, inter):
    cos, sin = rope_tables(rot, 5000, 1e4, device="cpu")
    fused = randn(rows, (heads + 1) * D, seed=rows + D, dtype=dtype)
    pos = torch.randint(0, 5000, (rows,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    x = fused[:, : heads * D].unflatten(1, (heads, D))
    want = R.turn(x, pos, cos, sin, inter)
    xd, c, s = fused.to(DEV)[:, : heads * D].unflatten(1, (heads, D)), cos.to(DEV), sin.to(DEV)
    got = rope(xd, pos.to(DEV), c, s, interleaved=inter)
    assert torch.equal(got.cpu(), want)
    # 64 bits: a table entry is off by half a step (2^-24 relative to at most 1), two products and a sum round once each, the result once to its type
    i = torch.arange(rot // 2, dtype=torch.float64)
    a = pos.double()[:, None] * 1e4 ** (-2 * i / rot)
    exact = x.double().clone()
    f, g = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    p, q = x.double()[..., f], x.double()[..., g]
    exact[..., f], exact[..., g] = p * a.cos()[:, None] - q * a.sin()[:, None], q * a.cos()[:, None] + p * a.sin()[:, None]
    size = torch.zeros_like(exact)
    size[..., f] = size[..., g] = p.abs() + q.abs()
    assert ((got.cpu().double() - exact).abs() <= 4 * 2.0**-24 * size + exact.abs() * torch.finfo(dtype).eps / 2 + 1e-30).all()
    # in place, rows that are not 16-byte aligned (the element-wise path), heads further apart than they are wide
    rope(xd, pos.to(DEV), c, s, interleaved=inter, out=xd)
    assert torch.equal(xd.cpu(), want)
    odd = torch.zeros(rows, heads, D + 3, dtype=dtype, device=DEV)[..., 1 : D + 1]
    odd.copy_(x)
    assert torch.equal(rope(odd, pos.to(DEV), c, s, interleaved=inter).cpu(), want)


def test_rope_leaves_negative_positions_and_marks_those_behind_the_table():
    cos, sin = rope_tables(32, 10, device=DEV)
    x = randn(4, 2, 64, seed=3).to(DEV)
    out = torch.full_like(x, 7.0)
    rope(x, i32([-1, 9, 10, 2**31 - 1]), cos, sin, out=out)
    assert (out[0] == 7).all() and torch.isfinite(out[1]).all()
    assert torch.isnan(out[2:, :, :32]).all() and torch.equal(out[2:, :, 32:], x[2:, :, 32:])
    assert rope(x[:0], i32([]), cos, sin).shape == (0, 2, 64)


# ---- append and read ------------------------------------------------------------------------------------------------------------------------

APPENDS = [  # new rows, rows before, Hkv, H, D, ps, rot, interleaved
    ([1], [0], 1, 1, 64, 64, 64, False),
    ([1, 1, 1, 1, 1], [0, 63, 64, 200, 7], 8, 16, 128, 64, 128, False),
    ([1, 0, 1], [130, 5, 127], 2, 14, 256, 128, 64, True),
    ([5, 0, 64, 1, 130], [60, 3, 0, 64, 1], 2, 4, 128, 64, 32, True),
    ([300, 17], [65, 1000], 3, 3, 64, 256, 64, False),
    ([9, 2], [2, 62], 1, 7, 256, 64, 256, False),
    ([33, 71, 8], [8, 24, 61], 4, 4, 128, 64, 10, False),  # rotary_dim not a multiple of 16: the element-wise path
]


@pytest.mark.parametrize("kind,dtype", [("model", F32), ("model", BF), ("int4", BF)])
@pytest.mark.parametrize("case", APPENDS)
def test_append_and_read(kind, dtype, case):
    new, past, Hkv, H, D, ps, rot, inter = case
    B, T, cu = len(new), sum(new), ragged(new)
    total = [p + n for p, n in zip(past, new)]
    table, n_pages = make_table(total, ps, 3, seed=T)
    cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    cos, sin = rope_tables(rot, max(total), 1e4, device="cpu")
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]) if T else torch.zeros(0)
    extra = 2  # rows behind the last session: read and written by nobody
    fused = randn(T + extra, (H + 2 * Hkv) * D, seed=T + D, dtype=dtype)
    rows = fused.to(DEV)
    q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([H * D, Hkv * D, Hkv * D], 1))
    q_out = torch.full((T + extra, H, D), 5.0, dtype=dtype, device=DEV)
    args = dict(max_new=max(new), cos=cos.to(DEV), sin=sin.to(DEV), interleaved=inter)
    tb, st, cud = table.to(DEV), i32(past), i32(cu)
    # what was there stays: write the earlier rows first where there are few
    before = None
    if max(past) <= 256:
        ck, cv = randn(sum(past), Hkv, D, seed=9, dtype=dtype).to(DEV), randn(sum(past), Hkv, D, seed=8, dtype=dtype).to(DEV)
        cache.append(ck, cv, tb, i32([0] * B), i32(ragged(past)), max_new=max(past + [1]))
        before = cache.read(tb, i32([0] * B), i32(ragged(past)), sum(past), max_new=max(past + [1]))
    got = cache.append(k, v, tb, st, cud, q=q, q_out=q_out, **args)
    assert got is q_out
    qw, kw = (R.turn(x.cpu()[:T], pos, cos, sin, inter) for x in (q, k))
    vw = v.cpu()[:T]
    assert torch.equal(q_out.cpu()[:T], qw) and (q_out[T:] == 5).all()
    if kind == "int4":
        kw, vw = R.four_bit_values(kw).to(BF), R.four_bit_values(vw).to(BF)
    rk, rv = cache.read(tb, st, cud, T, max_new=max(new))
    assert torch.equal(rk.cpu(), kw) and torch.equal(rv.cpu(), vw)
    if before is not None:
        again = cache.read(tb, i32([0] * B), i32(ragged(past)), sum(past), max_new=max(past + [1]))
        assert torch.equal(again[0], before[0]) and torch.equal(again[1], before[1])
    # pages of nobody are untouched
    used = set(table[table >= 0].tolist())
    for pg in set(range(n_pages)) - used:
        for t in (cache.k, cache.v, cache.k_meta, cache.v_meta):
            assert t is None or (t[pg].view(torch.uint8) == 255).all()
    # rows that are not 16-byte aligned take the element-wise path to the same bytes
    other = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    if before is not None:
        other.append(ck, cv, tb, i32([0] * B), i32(ragged(past)), max_new=max(past + [1]))
    odd = torch.zeros(T + extra, fused.shape[1] + 3, dtype=dtype, device=DEV)[:, 1 : 1 + fused.shape[1]]
    odd.copy_(rows)
    q2, k2, v2 = (x.unflatten(1, (-1, D)) for x in odd.split([H * D, Hkv * D, Hkv * D], 1))
    q2_out = other.append(k2, v2, tb, st, cud, q=q2, q_out=q2, **args)     # and queries in place
    assert torch.equal(q2_out.cpu()[:T], qw)
    for a, b in ((cache.k, other.k), (cache.v, other.v), (cache.k_meta, other.k_meta), (cache.v_meta, other.v_meta)):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("new,past", [([70], [30]), ([1, 1], [5, 64])])
def test_four_bit_pages_hold_what_the_layout_says(new, past):
    Hkv, D, ps = 2, 128, 64
    total = [p + n for p, n in zip(past, new)]
    table, n_pages = make_table(total, ps, 1, seed=4)
    cache = poisoned(n_pages, Hkv, D, ps, "int4")
    T = sum(new)
    k, v = randn(T, Hkv, D, seed=1, dtype=BF, scale=3), randn(T, Hkv, D, seed=2, dtype=BF)
    k[0, 0, :32] = 2.5        # a group without a range: scale 0, code 8
    k[0, 1, 5] = 1e30         # cut to 32768
    v[0, 0, 40] = float("inf")
    v[0, 1, 1] = float("nan")  # a group that holds no number reads as NaN
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32(past), i32(ragged(new)), max_new=max(new))
    kc, ks, kz = R.four_bits(k)
    vc, vs, vz = R.four_bits(v)
    i = 0
    for b, n in enumerate(new):
        for j in range(n):
            p = past[b] + j
            pg, at = int(table[b, p // ps]), p % ps
            assert torch.equal(R.page_key_codes(cache.k[pg].cpu())[:, at], kc[i])
            km = cache.k_meta[pg, :, at].cpu().float()
            assert torch.equal(km[..., 0], ks[i]) and torch.equal(km[..., 1], kz[i])
            vm = cache.v_meta[pg, :, :, :, at].cpu().float()
            got = R.page_value_codes(cache.v[pg].cpu())[:, at]
            for h in range(Hkv):
                for g in range(D // 32):
                    if torch.isfinite(v[i, h, 32 * g : 32 * g + 32]).all():
                        assert torch.equal(got[h, 32 * g : 32 * g + 32], vc[i, h, 32 * g : 32 * g + 32])
                        assert vm[h, g, 0] == vs[i, h, g] and vm[h, g, 1] == vz[i, h, g]
                    else:
                        assert vm[h, g, 0] == 0 and torch.isnan(vm[h, g, 1])
            i += 1
    rk, rv = cache.read(table.to(DEV), i32(past), i32(ragged(new)), T, max_new=max(new))
    assert (rk[0, 0, :32] == 2.5).all() and torch.isnan(rv[0, 0, 32:64]).all() and torch.isnan(rv[0, 1, :32]).all() and torch.isfinite(rv[0, 0, :32]).all()


def test_rows_without_a_page_are_not_stored_and_read_as_zero():
    Hkv, D, ps = 1, 64, 64
    cos, sin = rope_tables(64, 100, device=DEV)
    table = torch.tensor([[1, -1, 0], [5, 2, 3]], dtype=torch.int32)  # session 0 has a hole at 64 .. 127; page 5 does not exist
    for new, start in (([150, 100], [20, 30]), ([1, 1], [64, 10]), ([1, 1], [500, 2**31 - 1])):
        cache = poisoned(5, Hkv, D, ps, "model", F32)
        T = sum(new)
        k, v = randn(T, Hkv, D, seed=5).to(DEV), randn(T, Hkv, D, seed=6).to(DEV)
        cache.append(k, v, table.to(DEV), i32(start), i32(ragged(new)), max_new=max(new))
        rk, rv = cache.read(table.to(DEV), i32(start), i32(ragged(new)), T, max_new=max(new))
        i = 0
        for b in range(2):
            for j in range(new[b]):
                p = start[b] + j
                if p >= 2**31 - 1:
                    continue  # behind every table: left as it is
                pg = int(table[b, p // ps]) if p // ps < 3 else -1
                if 0 <= pg < 5:
                    assert torch.equal(rk[i], k[i]) and torch.equal(rv[i], v[i])
                else:
                    assert (rk[i] == 0).all() and (rv[i] == 0).all()
                i += 1
        assert torch.isnan(cache.k[4]).all() and torch.isnan(cache.v[4]).all()
    # keys behind the rotary tables are NaN in the channels that turn
    cache = poisoned(5, Hkv, D, ps, "model", F32)
    k = randn(2, Hkv, D, seed=5).to(DEV)
    t2 = i32([[0, 1], [2, 3]])
    cache.append(k, k, t2, i32([99, 100]), cos=cos[:, :16].contiguous(), sin=sin[:, :16].contiguous())
    rk, rv = cache.read(t2, i32([99, 100]))
    assert torch.isfinite(rk[0]).all() and torch.isnan(rk[1, :, :32]).all() and torch.equal(rk[1, :, 32:], k[1, :, 32:]) and torch.equal(rv, k)


# ---- attention --------------------------------------------------------------------------------------------------------------------------------


def tolerance(o, size, kind, dtype, vmax, S, D, split_probs):
    """How far the kernel may be from 64 bits, elementwise, from its roundings (all relative to |v| <= vmax, the weights summing to 1):
    a score's f32 dot product, scaling and maximum: (D + 4) half steps of f32 of sum |q k|; 4-bit keys: half a step of f16 more;
    exp2 (2 half steps) and a sum of S weights (S half steps, numerator and denominator); weights as product operands: half a step of bf16
    (2^-16 where the remainder is a second operand) or f16; 4-bit values: half a step of f16; the result: half a step of its type.
    An error e of a score moves the result by at most 2 e vmax."""
    u = 2.0**-24
    score = (D + 4) * u * size + (2.0**-11 * size if kind == "int4" else 0)
    weight = (2 * S + 8) * u + (2.0**-11 + 2.0**-11 if kind == "int4" else 0.0 if dtype == F32 else 2.0**-16 if split_probs else 2.0**-8)
    return (2 * score[..., None] + weight) * vmax * 1.01 + o.abs() * torch.finfo(dtype).eps / 2 + 1e-30


def check_attention(new, kv, Hkv, H, D, ps, kind, dtype, causal=True, window=0, seed=0, holes=(), scale=None, few=True, max_kv=None, aligned=True, amp=1.0):
    B, T, cu = len(new), sum(new), ragged(new)
    table, n_pages = make_table(kv, ps, 2, seed)
    cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
    S = sum(kv)
    k, v = randn(S, Hkv, D, seed=seed + 1, dtype=dtype, scale=amp), randn(S, Hkv, D, seed=seed + 2, dtype=dtype)
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32([0] * B), i32(ragged(kv)), max_new=max(kv + [1]))
    for b, c in holes:
        table[b, c] = -1 if (b + c) % 2 else n_pages + 3
    kd, vd = (R.four_bit_values(x).double() for x in (k, v)) if kind == "int4" else (k.double(), v.double())
    q = randn(T + 3, H, D, seed=seed + 3, dtype=dtype)
    qd, out = q.to(DEV), torch.full((T + 3, H, D), 3.0, dtype=dtype, device=DEV)
    if not aligned:
        qd, out = (torch.zeros(T + 3, H * D + 3, dtype=dtype, device=DEV)[:, 1 : 1 + H * D].unflatten(1, (H, D)).copy_(x) for x in (qd, out))
    got = cache.attend(qd, table.to(DEV), i32(kv), i32(cu), max_new=max(new + [1]), max_kv=max_kv if max_kv is not None else max(kv), causal=causal, window=window, out=out, scale=scale)
    assert got is out
    got, starts = out.cpu().double(), ragged(kv)
    assert (got[T:] == 3).all()
    for b in range(B):
        kk, vv = kd[starts[b] : starts[b + 1]], vd[starts[b] : starts[b + 1]]
        seen = torch.ones(kv[b], dtype=torch.bool)
        for bb, c in holes:
            if bb == b:
                seen[c * ps : (c + 1) * ps] = False
        want, size = R.attend(q[cu[b] : cu[b + 1]].double(), kk, vv, new[b], D**-0.5 if scale is None else scale, causal, window, seen)
        # the second operand goes with the kernel for at most 32 (row, head) pairs per KV head; above that the weights are one bf16 operand: each is off by
        # half a step, 2^-8 of itself, and sum p |v| <= vmax
        tol = tolerance(want, size, kind, dtype, float(vv.abs().max()) if kv[b] else 0.0, kv[b], D, few and max(new) * (H // Hkv) <= 32)
        err = (got[cu[b] : cu[b + 1]] - want).abs()
        assert (err <= tol).all(), (b, float((err / tol).max()), float(err.max()))
    return cache, table


KINDS = [("model", F32), ("model", BF), ("int4", BF)]
STEPS = [  # positions of every session, Hkv, H, D, ps: one new row each
    ([1], 1, 1, 64, 64),
    ([203], 8, 16, 128, 64),
    ([1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129], 2, 4, 64, 64),
    ([0, 257, 1000, 5], 3, 3, 128, 128),
    ([700, 1, 64], 2, 14, 256, 64),
    ([5000, 17], 1, 20, 64, 256),
    ([3001], 2, 2, 128, 1024),
    ([300, 299], 1, 40, 128, 64),
]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("kv,Hkv,H,D,ps", STEPS)
def test_attend_one_row_per_session(kind, dtype, kv, Hkv, H, D, ps):
    check_attention([1] * len(kv), kv, Hkv, H, D, ps, kind, dtype)
    check_attention([1] * len(kv), kv, Hkv, H, D, ps, kind, dtype, causal=False, seed=7, aligned=False, max_kv=-(-max(kv) // ps) * ps)
    check_attention([1] * len(kv), kv, Hkv, H, D, ps, kind, dtype, window=70, seed=9, amp=4.0)


PROMPTS = [  # new rows, positions with them, Hkv, H, D, ps
    ([2, 3], [2, 70], 1, 2, 64, 64),
    ([40, 0, 65], [40, 9, 300], 2, 4, 128, 64),
    ([130, 7], [129, 3], 2, 2, 64, 64),          # more new rows than positions: the first rows see nothing
    ([257], [600], 1, 7, 128, 128),
    ([20, 100], [700, 0], 1, 1, 256, 64),
    ([300, 129, 1], [300, 1500, 1200], 4, 4, 64, 64),
    ([33, 150], [33, 190], 1, 20, 64, 256),
]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,kv,Hkv,H,D,ps", PROMPTS)
def test_attend_prompts(kind, dtype, new, kv, Hkv, H, D, ps):
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, few=False)
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, causal=False, seed=3, few=False, aligned=False)
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, window=50, seed=5, few=False)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_attend_many_sessions_with_prompts(kind, dtype):
    """More sessions than are sorted by length (64), exactly as many, and pair counts that are and are not a multiple of 8."""
    r = random.Random(5)
    for B, Hkv in ((70, 2), (64, 1), (65, 1), (13, 8)):
        kv = [r.choice([0, 1, 40, 64, 100, 333]) for _ in range(B)]
        new = [r.choice([0, 1, 2, 33, 70]) for _ in range(B)]
        check_attention(new, kv, Hkv, 2 * Hkv, 64, 64, kind, dtype, seed=B, few=False)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("B,Hkv,new", [(33, 8, 5), (64, 5, 5), (65, 5, 5)])
def test_attend_ragged_sessions_over_long_tables(kind, dtype, B, Hkv, new):
    """More workgroups than CUs and tables of 1024 positions and more: sessions are taken by length up to 64 of them, some without rows or positions."""
    r = random.Random(B)
    kv = [r.choice([0, 1, 64, 130, 700, 1100]) for _ in range(B - 1)] + [1100]
    rows = [r.choice([0, 1, new]) for _ in range(B - 1)] + [new]
    check_attention(rows, kv, Hkv, Hkv * 13, 64, 64, kind, dtype, seed=B, few=False)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("new,kv,Hkv,H,D,ps", [([40], [4100], 1, 2, 64, 64), ([70, 3], [2500, 3], 1, 1, 128, 128), ([35], [1300], 1, 2, 256, 64)])
def test_attend_few_rows_of_a_long_past_in_splits(kind, dtype, new, kv, Hkv, H, D, ps):
    """A few tiles of rows over thousands of positions: many splits, some of them behind every row or empty."""
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, few=False)
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, causal=False, seed=3, few=False, aligned=False, max_kv=-(-max(kv) // ps) * ps)
    check_attention(new, kv, Hkv, H, D, ps, kind, dtype, window=700, seed=5, few=False)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("rows", [17, 24, 32, 33, 64, 65])
def test_attend_row_counts_around_the_kernels_borders(kind, dtype, rows):
    """(row, head) pairs per KV head at which one kernel hands over to the other, with few and with many sessions."""
    check_attention([rows, 1], [200, 77], 1, 1, 64, 64, kind, dtype, seed=rows, few=False)
    check_attention([1] * 5, [70, 1, 300, 64, 2], 1, rows, 128, 64, kind, dtype, seed=rows, few=False)
    check_attention([rows // 8] * 40, [rows // 8 + 7 * (i % 9) for i in range(40)], 8, 64, 64, 64, kind, dtype, seed=rows, few=False)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_attend_skips_positions_without_a_page(kind, dtype):
    check_attention([1, 1], [500, 300], 2, 4, 128, 64, kind, dtype, holes=[(0, 0), (0, 3), (1, 4)])
    check_attention([1], [64], 2, 4, 64, 64, kind, dtype, holes=[(0, 0)])      # nothing left: zero
    check_attention([90, 200], [500, 300], 1, 4, 64, 64, kind, dtype, holes=[(0, 2), (1, 0), (1, 1)], few=False)


def test_attend_values_that_only_other_rows_see():
    """A NaN behind kv_len, in front of every row's window and behind the last page's end stays out of the result."""
    Hkv, D, ps = 1, 64, 64
    for kind, dtype in KINDS:
        table, n = make_table([190], ps, 0, 1)
        cache = poisoned(n, Hkv, D, ps, kind, dtype)
        k, v = randn(190, Hkv, D, seed=1, dtype=dtype), randn(190, Hkv, D, seed=2, dtype=dtype)
        k[:100], v[:100] = float("nan"), float("nan")
        cache.append(k.to(DEV), v.to(DEV), table.to(DEV), i32([0]), i32([0, 190]), max_new=190)
        for new, kv, window in ((1, 150, 50), (30, 160, 31), (1, 101, 1)):
            q = randn(new, 2, D, seed=3, dtype=dtype).to(DEV)
            o = cache.attend(q, table.to(DEV), i32([kv]), i32([0, new]), max_new=new, window=window)
            assert torch.isfinite(o).all(), (kind, new)


def test_attend_with_scores_far_apart_and_infinite():
    """Scores of +-1e4: the maximum is subtracted before anything is exponentiated; a score of -inf counts nothing."""
    for kind, dtype in KINDS:
        check_attention([1, 40], [333, 200], 1, 2, 128, 64, kind, dtype, amp=100.0, scale=1.0, few=False)
    cache = poisoned(2, 1, 64, 64, "model", F32)
    k, v = randn(70, 1, 64, seed=1), randn(70, 1, 64, seed=2)
    k[3:60, 0, 0], k[:, 0, 1:] = -float("inf"), 0.0
    table = i32([[1, 0]])
    cache.append(k.to(DEV), v.to(DEV), table, i32([0]), i32([0, 70]), max_new=70)
    q = torch.zeros(1, 1, 64)
    q[..., 0] = 1.0
    o = cache.attend(q.to(DEV), table, i32([70]), causal=False).cpu()
    keep = torch.tensor([i for i in range(70) if not 3 <= i < 60])
    p = torch.softmax(k[keep, 0, 0].double() / 8, 0)
    assert (o[0, 0].double() - p @ v[keep, 0].double()).abs().max() < 1e-5


def test_attend_keeps_a_long_tail_of_small_weights():
    """One position with nearly all the weight and 60000 of 2^-29 to 2^-25 of it whose values point the same way: together 1e-4 to 2e-3 of the result, which float16 weights
    below 2^-24 of the largest would drop."""
    Hkv, D, ps, n = 1, 64, 64, 60000
    table, n_pages = make_table([n], ps, 0, 1)
    for kind, dtype in KINDS:
        for tail in (-29, -27, -25):
            cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
            k, v = torch.zeros(n, Hkv, D), torch.ones(n, Hkv, D)
            k[0, 0, :32], v[0] = 1.0, 0.0
            cache.append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), table.to(DEV), i32([0]), i32([0, n]), max_new=n)
            for rows in (1, 70):
                q = torch.full((rows, 1, D), 1.0, dtype=dtype, device=DEV)
                scale = -tail / 32 * 0.6931471805599453
                o = cache.attend(q, table.to(DEV), i32([n]), i32([0, rows]), max_new=rows, causal=False, scale=scale).cpu().double()
                w = (n - 1) * 2.0**tail
                want = w / (1 + w)
                # the score of position 0 is exact up to its f32 product (2^-22 of |tail|), a weight is off by half a step of its type (2^-8 at most), and of float16 by
                # 2^-25 of 2^-7 of the largest at most; the sums of n weights in f32 by n half steps at worst
                tol = want * (2.0**-8 + abs(tail) * 2.0**-21 + n * 2.0**-24) + (n * 2.0**-32 if kind == "int4" else 0) + want * torch.finfo(dtype).eps / 2
                assert (o - want).abs().max() <= tol, (kind, dtype, tail, rows, float((o - want).abs().max() / want))


def test_offsets_behind_32_bits():
    """Pages whose elements (and bytes) lie behind 2^32, and a row buffer just as long."""
    for kind, dtype, n_pages in (("model", BF, 34000), ("int4", BF, 70000)):
        Hkv, D, ps = 8, 256, 64
        cache = PagedKVCache(n_pages, Hkv, D, page_size=ps, kind=kind, dtype=dtype, device=DEV)
        assert cache.k.numel() > 2**32
        table = i32([[n_pages - 1, 0, n_pages - 2], [n_pages // 2, n_pages - 3, 1]])
        new = [150, 140]
        k, v = randn(290, Hkv, D, seed=1, dtype=dtype), randn(290, Hkv, D, seed=2, dtype=dtype)
        cache.append(k.to(DEV), v.to(DEV), table, i32([0, 0]), i32([0, 150, 290]), max_new=150)
        rk, rv = cache.read(table, i32([0, 0]), i32([0, 150, 290]), 290, max_new=150)
        kw, vw = (R.four_bit_values(x).to(BF) for x in (k, v)) if kind == "int4" else (k, v)
        assert torch.equal(rk.cpu(), kw) and torch.equal(rv.cpu(), vw)
        kd, vd = (R.four_bit_values(x).double() for x in (k, v)) if kind == "int4" else (k.double(), v.double())
        q = randn(2, Hkv, D, seed=3, dtype=dtype)
        o = cache.attend(q.to(DEV), table, i32(new), max_kv=150).cpu().double()
        for b, (lo, hi) in enumerate(((0, 150), (150, 290))):
            want, size = R.attend(q[b : b + 1].double(), kd[lo:hi], vd[lo:hi], 1, D**-0.5)
            assert ((o[b : b + 1] - want).abs() <= tolerance(want, size, kind, dtype, float(vd.abs().max()), 150, D, True)).all()
        del cache


# ---- as they are used together ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_a_serving_loop(kind, dtype):
    """Prompts of three sessions, then steps in which one session pauses and another gets a further turn: against plain attention over the whole past."""
    Hkv, H, D, ps, rot = 2, 6, 64, 64, 32
    cos, sin = rope_tables(rot, 512, 1e4, scaling="yarn", factor=2.0, original=128, device="cpu")
    c, s = cos.to(DEV), sin.to(DEV)
    table, n_pages = make_table([400, 400, 400], ps, 1, 3)
    cache, tb = poisoned(n_pages, Hkv, D, ps, kind, dtype), table.to(DEV)
    have, past_k, past_v = [0, 0, 0], [[], [], []], [[], [], []]
    turns = [[70, 1, 33], [1, 1, 1], [1, 0, 1], [1, 90, 1], [1, 1, 1], [1, 1, 1]]
    for step, new in enumerate(turns):
        T, cu = sum(new), ragged(new)
        q, k, v = (randn(T, h, D, seed=100 * step + h, dtype=dtype) for h in (H, Hkv, Hkv + 100))
        v = v[:, :Hkv].contiguous()
        args = dict(max_new=max(new))
        qt = cache.append(k.to(DEV), v.to(DEV), tb, i32(have), i32(cu), cos=c, sin=s, q=q.to(DEV), **args)
        pos = torch.cat([torch.arange(h, h + n) for h, n in zip(have, new)])
        kt, qw = R.turn(k, pos, cos, sin, False), R.turn(q, pos, cos, sin, False)
        assert torch.equal(qt.cpu(), qw)
        have = [h + n for h, n in zip(have, new)]
        o = cache.attend(qt, tb, i32(have), i32(cu), max_kv=max(have), **args).cpu().double()
        kt, vt = (R.four_bit_values(kt).double(), R.four_bit_values(v).double()) if kind == "int4" else (kt.double(), v.double())
        for b in range(3):
            past_k[b].append(kt[cu[b] : cu[b + 1]])
            past_v[b].append(vt[cu[b] : cu[b + 1]])
            kk, vv = torch.cat(past_k[b]), torch.cat(past_v[b])
            want, size = R.attend(qw[cu[b] : cu[b + 1]].double(), kk, vv, new[b], D**-0.5)
            tol = tolerance(want, size, kind, dtype, float(vv.abs().max()), len(kk), D, False)
            assert ((o[cu[b] : cu[b + 1]] - want).abs() <= tol).all(), (step, b)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_captured_step_replays_with_other_lengths(kind, dtype):
    """One decode step in a graph, its own workspace, replayed while the lengths on the device grow: every replay against the eager call."""
    Hkv, H, D, ps, B = 2, 4, 128, 64, 3
    cos, sin = rope_tables(D, 2048, device=DEV)
    table, n_pages = make_table([2000] * B, ps, 0, 5)
    tb = table.to(DEV)
    past = [900, 63, 1]
    kr, vr = randn(sum(past), Hkv, D, seed=1, dtype=dtype).to(DEV), randn(sum(past), Hkv, D, seed=2, dtype=dtype).to(DEV)
    caches = [poisoned(n_pages, Hkv, D, ps, kind, dtype) for _ in range(2)]
    for c in caches:
        c.append(kr, vr, tb, i32([0] * B), i32(ragged(past)), max_new=max(past), cos=cos, sin=sin)
    start, kv = i32(past), i32([p + 1 for p in past])
    q, k, v = (torch.zeros(B, h, D, dtype=dtype, device=DEV) for h in (H, Hkv, Hkv))
    ws = torch.empty(caches[0].workspace_bytes(H, B, B, max_kv=2000), dtype=torch.uint8, device=DEV)
    assert ws.numel() > 0  # the lengths are split: the second kernel is in the graph too
    out, qt = torch.empty_like(q), torch.empty_like(q)

    def step(c, out, qt):
        c.append(k, v, tb, start, cos=cos, sin=sin, q=q, q_out=qt)
        c.attend(qt, tb, kv, max_kv=2000, out=out, workspace=ws)

    step(caches[0], out, qt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(caches[0], out, qt)
    for i in range(5):
        q.copy_(randn(B, H, D, seed=50 + i, dtype=dtype))
        k.copy_(randn(B, Hkv, D, seed=60 + i, dtype=dtype))
        v.copy_(randn(B, Hkv, D, seed=70 + i, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        want, wq = torch.empty_like(q), torch.empty_like(q)
        step(caches[1], want, wq)
        torch.cuda.synchronize()
        assert torch.equal(qt, wq) and torch.equal(out, want), i
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        start += 1
        kv += 1


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_queries_in_place_and_a_captured_prompt(kind, dtype):
    """Appending with queries turned in place gives the rows of the call with a buffer for them; the prompt in a graph gives the eager result, replay after replay."""
    Hkv, H, D, ps = 2, 4, 128, 64
    cos, sin = rope_tables(64, 512, device=DEV)
    for new, past in (([1, 1, 1], [5, 64, 200]), ([90, 3, 41], [0, 64, 100])):
        T, cu, total = sum(new), i32(ragged(new)), [a + b for a, b in zip(new, past)]
        table, n_pages = make_table(total, ps, 0, T)
        tb, start, kv = table.to(DEV), i32(past), i32(total)
        cache = poisoned(n_pages, Hkv, D, ps, kind, dtype)
        kp, vp = randn(sum(past), Hkv, D, seed=1, dtype=dtype).to(DEV), randn(sum(past), Hkv, D, seed=2, dtype=dtype).to(DEV)
        cache.append(kp, vp, tb, i32([0] * 3), i32(ragged(past)), max_new=max(past))
        q, k, v = (torch.zeros(T, h, D, dtype=dtype, device=DEV) for h in (H, Hkv, Hkv))
        args = dict(max_new=max(new), cos=cos, sin=sin)
        out = torch.empty_like(q)

        def turn():
            w = cache.append(k, v, tb, start, cu, q=q, **args)
            cache.attend(w, tb, kv, cu, max_new=max(new), max_kv=max(total), out=out)
            return w

        turn()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            turned = turn()
        for i in range(3):
            for t, s in ((q, 10), (k, 20), (v, 30)):
                t.copy_(randn(*t.shape, seed=s + i, dtype=dtype))
            graph.replay()
            torch.cuda.synchronize()
            replayed, was = out.clone(), turned.clone()
            out.zero_()
            again = turn()
            torch.cuda.synchronize()
            assert torch.equal(again, was) and torch.equal(out, replayed)
            inplace = q.clone()
            assert cache.append(k, v, tb, start, cu, q=inplace, q_out=inplace, **args) is inplace
            assert torch.equal(inplace, was)


def test_other_streams_and_repeated_calls_agree():
    Hkv, H, D, ps = 2, 8, 128, 64
    kv = [1900, 700, 64, 1]
    cache, table = check_attention([1] * 4, kv, Hkv, H, D, ps, "int4", BF)
    tb, lens = table.to(DEV), i32(kv)
    q = randn(4, H, D, seed=1, dtype=BF).to(DEV)
    want = cache.attend(q, tb, lens, max_kv=1900)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(cache.attend(q, tb, lens, max_kv=1900))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
