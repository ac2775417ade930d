"""The paged cache's operators without a GPU: tables, refusals of the C ABI and of the Python entry points (nothing is launched)."""

import ctypes as C
import math

import pytest
import torch

from speech_to_speech_amd import native, paged_kv
from speech_to_speech_amd.paged_kv import PagedKVCache, rope, rope_frequencies, rope_tables

P = 0x1000  # a pointer nothing follows: every call below is refused before a launch


def handle(**kw):
    f = dict(k=P, v=P, k_meta=0, v_meta=0, n_pages=4, page_size=64, kv_heads=2, head_dim=128, kind=0, dtype=native.S2S_BF16)
    f.update(kw)
    return native.PagedKVStruct(*(f[n] for n, _ in native.PagedKVStruct._fields_))


def attend(kv, *, ws=0, ws_bytes=0, H=4, cols=8, cu=0, B=1, T=1, max_new=1, max_kv=512, causal=1, window=0, q=P, lens=P, table=P):
    return native.load().s2s_op_attn_paged(None, C.byref(kv) if kv else None, q, H * 128, P, H * 128, H, table, cols, lens, cu, B, T, max_new, max_kv, 1.0, causal, window, ws, ws_bytes)


def append(kv, *, q=0, q_out=0, H=0, cols=8, cu=0, B=1, T=1, max_new=1, cos=P, sin=P, max_pos=10, rot=128, k=P, table=P, start=P):
    return native.load().s2s_op_kv_append_paged(None, C.byref(kv), k, 256, P, 256, q, H * 128, q_out, H * 128, H, table, cols, start, cu, B, T, max_new, cos, sin, max_pos, rot, 0)


@pytest.mark.parametrize("kv,word", [(dict(head_dim=96), b"head_dim"), (dict(page_size=96), b"page_size"), (dict(page_size=32), b"page_size"), (dict(page_size=2048), b"page_size"),
                                     (dict(n_pages=0), b"pages"), (dict(kv_heads=0), b"heads"), (dict(k=0), b"missing"), (dict(v=P + 8), b"aligned"), (dict(kind=7), b"kind"),
                                     (dict(dtype=5), b"dtype"), (dict(kind=1), b"k_meta"), (dict(kind=1, k_meta=P, v_meta=P, dtype=0), b"bf16")])
def test_bad_caches_are_refused(kv, word):
    lib = native.load()
    h = handle(**kv)
    for st in (attend(h), append(h), lib.s2s_op_kv_read_paged(None, C.byref(h), P, 8, P, 0, 1, 1, 1, P, P, 256), lib.s2s_op_attn_paged_ws(C.byref(h), 4, 1, 1, 1, 512, 1, 0)):
        assert st == -1
        assert word in lib.s2s_last_error()


def test_bad_calls_are_refused():
    lib, kv = native.load(), handle()
    assert attend(None) == -1
    for kw in (dict(H=3), dict(H=0), dict(window=5, causal=0), dict(window=-1), dict(max_kv=513), dict(max_kv=-1), dict(T=2), dict(max_new=2), dict(max_new=0), dict(cols=0),
               dict(q=0), dict(lens=0), dict(table=0), dict(B=-1, T=-1), dict(B=65536, T=65536), dict(cols=2**26)):
        assert attend(kv, **kw) == -1, kw
    # long pasts of few sessions are split: without a workspace, or with one too small or not aligned, the call is refused
    need = lib.s2s_op_attn_paged_ws(C.byref(kv), 4, 1, 1, 1, 65536, 1, 0)
    assert need > 0
    for ws, n in ((0, 0), (0, need), (P, need - 1), (P + 4, need)):
        assert attend(kv, cols=1024, max_kv=65536, ws=ws, ws_bytes=n) == -1
        assert b"workspace" in lib.s2s_last_error()
    assert lib.s2s_op_attn_paged_ws(C.byref(kv), 4, 0, 0, 1, 512, 1, 0) == 0
    # more workgroups than a launch takes, more (row, head) pairs than an index holds
    assert attend(handle(kv_heads=1024), H=1024, cu=P, B=60000, T=2**26, max_new=2**26) == -1 and b"too many" in lib.s2s_last_error()
    assert attend(handle(kv_heads=1024), H=4096, cu=P, B=1, T=2**20, max_new=1) == -1 and b"too many" in lib.s2s_last_error()
    for kw in (dict(rot=0), dict(rot=129), dict(rot=130), dict(max_pos=0), dict(sin=0), dict(q=P), dict(q=P, q_out=P), dict(q=P, q_out=P, H=4, cos=0, sin=0), dict(k=0), dict(start=0),
               dict(table=0), dict(T=3), dict(max_new=4)):
        assert append(kv, **kw) == -1, kw
    rp = lambda **k: lib.s2s_op_rope(None, k.get("x", P), 128, 64, k.get("out", 2 * P), k.get("o_rs", 128), 64, k.get("pos", P), k.get("cos", P), P, k.get("max_pos", 5),  # noqa: E731
                                     k.get("rows", 3), k.get("heads", 2), k.get("D", 64), k.get("rot", 64), 0, k.get("dtype", 0))
    for kw in (dict(dtype=9), dict(rot=65), dict(rot=66), dict(rot=0), dict(D=2048), dict(rows=-1), dict(max_pos=0), dict(cos=0), dict(pos=0), dict(x=0), dict(out=P, o_rs=256),
               dict(rows=2**31 - 1)):
        assert rp(**kw) == -1, kw
    # no rows, no launch
    assert rp(rows=0) == 0 and rp(heads=0) == 0
    assert attend(kv, B=0, T=0) == 0 and append(kv, B=0, T=0) == 0 and attend(kv, cu=P, B=3, T=0) == 0


def test_python_entry_points_refuse_what_does_not_fit():
    c = PagedKVCache(4, 2, 64, device="cpu")
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table = i(0, 1, 2, 3).view(2, 2)
    rows = lambda h=2, n=2, d=64, dt=torch.bfloat16: torch.zeros(n, h, d, dtype=dt)  # noqa: E731
    cos, sin = rope_tables(64, 8, device="cpu")
    bad = [lambda: c.append(rows(3), rows(), table, i(0, 0)), lambda: c.append(rows(), rows(d=32), table, i(0, 0)), lambda: c.append(rows(dt=torch.float32), rows(), table, i(0, 0)),
           lambda: c.append(rows(), rows(), table.long(), i(0, 0)), lambda: c.append(rows(), rows(), table, i(0)), lambda: c.append(rows(), rows(n=1), table, i(0, 0)),
           lambda: c.append(rows(n=3), rows(n=3), table, i(0, 0)), lambda: c.append(rows(), rows(), table, i(0, 0), i(0, 1)), lambda: c.append(rows(), rows(), table, i(0, 0), q=rows(4)),
           lambda: c.append(rows(), rows(), table, i(0, 0), cos=cos), lambda: c.append(rows(), rows(), table, i(0, 0), cos=cos.double(), sin=sin.double()),
           lambda: c.append(torch.zeros(2, 64, 2, dtype=torch.bfloat16).transpose(1, 2), rows(), table, i(0, 0)),
           lambda: c.append(rows(), rows(), table, i(0, 0), cos=cos, sin=sin, q=rows(4), q_out=rows(3)), lambda: c.attend(rows(4, 2, 32), table, i(1, 1)),
           lambda: c.attend(rows(4), table, i(1, 1), out=rows(4, 3)), lambda: c.attend(rows(4), table, i(1, 1), max_new=2), lambda: c.attend(rows(4), table, i(1, 1), max_kv=129), lambda: c.attend(rows(4), table, i(1, 1), max_kv=2**32), lambda: c.read(table, i(0, 0), i(0, 1, 2)),
           lambda: rope(rows(), i(0), cos, sin), lambda: rope(rows(), i(0, 1), cos, sin[:4]), lambda: rope(rows(), i(0, 1), cos, sin, out=rows(3)),
           lambda: PagedKVCache(4, 2, 64, kind="int3", device="cpu"), lambda: PagedKVCache(4, 2, 64, kind="int4", dtype=torch.float32, device="cpu"),
           lambda: PagedKVCache.adopt(c.k, c.k[:3]), lambda: PagedKVCache.adopt(c.k, c.v, c.k), lambda: rope_tables(7, 4, device="cpu"), lambda: rope_tables(8, 4, scaling="odd", device="cpu"),
           lambda: rope_tables(8, 4, scaling="yarn", device="cpu"), lambda: rope_tables(2, 4, scaling="ntk", factor=2.0, device="cpu")]
    for f in bad:
        with pytest.raises((ValueError, native.NativeError)):
            f()
    # all in order, but there is no GPU behind these tensors: refused, not computed elsewhere
    for f in (lambda: c.append(rows(), rows(), table, i(0, 0)), lambda: c.attend(rows(4), table, i(1, 1)), lambda: c.read(table, i(0, 0)), lambda: rope(rows(), i(0, 1), cos, sin)):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_scaled_frequencies():
    d, theta = 64, 1e4
    plain = [theta ** (-2 * i / d) for i in range(d // 2)]
    w, m = rope_frequencies(d, theta)
    assert m == 1 and all(math.isclose(a, b, rel_tol=1e-14) for a, b in zip(w.tolist(), plain))
    w, m = rope_frequencies(d, theta, "linear", 4.0)
    assert m == 1 and all(math.isclose(a, b / 4, rel_tol=1e-14) for a, b in zip(w.tolist(), plain))
    w, m = rope_frequencies(d, theta, "ntk", 4.0)     # the fastest pair is kept, the slowest stretched by the factor
    assert m == 1 and w[0] == 1 and math.isclose(w[-1], plain[-1] / 4, rel_tol=1e-12)
    w, m = rope_frequencies(d, theta, "yarn", 4.0, 4096)
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    for a, b in zip(w.tolist(), plain):
        turns = 4096 * b / (2 * math.pi)
        if turns > 40:
            assert math.isclose(a, b, rel_tol=1e-12)
        elif turns < 0.7:
            assert math.isclose(a, b / 4, rel_tol=1e-12)
        else:
            assert b / 4 * (1 - 1e-12) <= a <= b * (1 + 1e-12)


def test_tables_hold_far_angles():
    cos, sin = rope_tables(8, 100001, 1e4, device="cpu")
    for p in (0, 1, 99999, 100000):
        for i in range(4):
            a = math.fmod(p * 1e4 ** (-i / 4), 2 * math.pi)
            assert abs(float(cos[p, i]) - math.cos(a)) < 2.0**-24 + 1e-10 and abs(float(sin[p, i]) - math.sin(a)) < 2.0**-24 + 1e-10
