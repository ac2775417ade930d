"""Measured work: rotary positions, the paged key / value cache and the attention that reads it.

Every case is one pass through one operator: ``run`` makes it in elementary torch operations in 32 bits, or - with ``own`` set -
through the framework's entry points (``speech_to_speech_amd.paged_kv``).

Layout of the cache, which both forms share.  A page holds ``ps`` positions of every KV head:

* keys ``[page][Hkv][ps][D]``, values transposed ``[page][Hkv][D][ps]`` in the model type;
* 4 bits: groups of 32 channels of one position, value = zero + scale * (code - 8), scale and zero in float16.  Codes of 8 neighbours (an
  octet: 8 channels of a key, 8 positions of a value channel) share 4 bytes, element e in nibble (e >> 1) + 4 * (e & 1).  Keys
  ``[page][Hkv][ps][D / 2]``: dword g * (D / 32) + s of a row holds channels 32 s + 8 g ...; values ``[page][Hkv][D][ps / 2]``, octets in
  order.  Scales and zeros: keys ``[page][Hkv][ps][D / 32][2]``, values ``[page][Hkv][D / 32][2][ps]``.
"""

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32, "int4": torch.bfloat16}


def listed():
    rope = {"op": "rope", "D": 128, "theta": 1e6}
    talker = {"H": 16, "Hkv": 8, "D": 128, "ps": 64}
    app = {"op": "append", "rot": 128, "inter": False, "theta": 1e6, **talker}
    att = {"op": "attend", "causal": True, "window": 0, **talker}
    return [
        # one frame of 64 speaking sessions: the talker's 16 query heads, still inside the fused projection's rows
        {"name": "rope_step", **rope, "dtype": "bf16", "heads": 16, "T": 64, "rot": 128, "inter": False, "scaling": "none", "factor": 1.0, "orig": 0, "max_pos": 4096},
        # a float32 engine's prompts: half of each head turns, neighbours are paired, positions stretched 4 x past the trained 32 k
        {"name": "rope_prompt", **rope, "dtype": "f32", "heads": 20, "T": 20011, "rot": 64, "inter": True, "scaling": "yarn", "factor": 4.0, "orig": 32768, "max_pos": 131072},
        # one frame of 64 sessions: a row each behind what their pages hold
        {"name": "append_step", **app, "kind": "bf16", "B": 64, "new_lo": 1, "new_hi": 1, "start_lo": 100, "start_hi": 1500},
        # the prompts of 24 sessions at once, some behind an earlier turn
        {"name": "append_prompt", **app, "kind": "bf16", "B": 24, "new_lo": 37, "new_hi": 2048, "start_lo": 0, "start_hi": 700},
        # the widest frame loop (512 sessions) over 4-bit pages, and the rows as the pages hold them
        {"name": "append4_step", **app, "kind": "int4", "B": 512, "new_lo": 1, "new_hi": 1, "start_lo": 100, "start_hi": 1500},
        # prompts into 4-bit pages
        {"name": "append4_prompt", **app, "kind": "int4", "B": 24, "new_lo": 37, "new_hi": 2048, "start_lo": 0, "start_hi": 700},
        # a single session of a float32 engine: the smallest call, where latency counts
        {"name": "attend_single", **att, "kind": "f32", "B": 1, "new_lo": 1, "new_hi": 1, "kv_lo": 203, "kv_hi": 203},
        # the widest frame loop: 512 sessions of ragged lengths
        {"name": "attend_step", **att, "kind": "bf16", "B": 512, "new_lo": 1, "new_hi": 1, "kv_lo": 61, "kv_hi": 1531},
        # ragged prompts, some behind an earlier turn of the same session
        {"name": "attend_prompt", **att, "kind": "bf16", "B": 8, "new_lo": 301, "new_hi": 4096, "kv_lo": 700, "kv_hi": 6001},
        # the encoder's 1500 frames of 64 sessions, read by one token each: no mask, a key head for every query head
        {"name": "attend4_cross", **att, "kind": "int4", "B": 64, "new_lo": 1, "new_hi": 1, "kv_lo": 1500, "kv_hi": 1500, "H": 20, "Hkv": 20, "D": 64, "causal": False},
        # few sessions with a long past
        {"name": "attend4_long", **att, "kind": "int4", "B": 7, "new_lo": 1, "new_hi": 1, "kv_lo": 9001, "kv_hi": 100021},
        # a further turn of 16 sessions over what they have said and heard so far
        {"name": "attend4_prompt", **att, "kind": "int4", "B": 16, "new_lo": 17, "new_hi": 401, "kv_lo": 900, "kv_hi": 4100},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "attend", "attend", "attend"])
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8, 20])
    H = Hkv * (1 if Hkv == 20 else rng.choice([1, 2, 4, 7]))
    inter = rng.random() < 0.4
    rot = rng.choice([D, D, D // 2, D // 4])
    ps = rng.choice([64, 64, 128])
    if op == "rope":
        heads = rng.randint(1, 32)
        T = _log(rng, 1, 20000 * 20 * 128 // (heads * D))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": op, "dtype": rng.choice(["bf16", "f32"]), "T": min(T, 60000), "heads": heads, "D": D, "rot": rot, "inter": inter,
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), "orig": 16384, "max_pos": 131072,
                "theta": rng.choice([1e4, 1e6])}
    kind = rng.choice(["bf16", "f32", "int4", "int4"])
    step = rng.random() < 0.55
    if op == "append":
        B = _log(rng, 1, 512) if step else _log(rng, 1, 24)
        hi = 1 if step else _log(rng, 2, max(2, min(4096, 24 * 2048 * 4 // (B * Hkv * max(1, D // 128)))))
        return {"op": op, "kind": kind, "B": B, "new_lo": 1 if step else max(1, hi // 5), "new_hi": hi, "start_lo": 0,
                "start_hi": _log(rng, 1, 1000), "H": H, "Hkv": Hkv, "D": D, "ps": ps, "rot": rot, "inter": inter, "theta": rng.choice([1e4, 1e6])}
    causal = rng.random() < 0.7
    wide = 2 if kind == "f32" else 1
    if step:
        B = _log(rng, 1, 512)
        new, kv = 1, _log(rng, 1, max(2, min(60000, 512 * 1500 * 8 * 128 // (2 * B * Hkv * D * wide))))
    else:
        B = _log(rng, 1, 16)
        kv = _log(rng, 16, 6000)
        new = max(1, min(kv, _log(rng, 2, 4096), int(8 * 4096 * 6000 * 16 * 128 / (4 * wide * B * kv * H * D))))
    return {"op": op, "kind": kind, "B": B, "new_lo": max(1, new // 3), "new_hi": new, "kv_lo": max(1, kv // 4), "kv_hi": kv, "H": H, "Hkv": Hkv,
            "D": D, "ps": ps, "causal": causal, "window": rng.choice([0, 0, 500]) if causal else 0}


def _spread(n, lo, hi, turn):
    """n lengths between lo and hi, each bound among them, in no order."""
    if n == 1:
        return [hi]
    return [lo, hi] + [lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + turn) % 1.0)) for i in range(1, n - 1)]


def _lengths(case):
    """New rows, and the rows in the cache behind them and with them, of every session."""
    new = _spread(case["B"], case["new_lo"], case["new_hi"], 0.37)
    if case["op"] == "append":
        start = _spread(case["B"], case["start_lo"], case["start_hi"], 0.11)[::-1]
        return new, start, [s + n for s, n in zip(start, new)]
    kv = [max(k, n) for k, n in zip(_spread(case["B"], case["kv_lo"], case["kv_hi"], 0.11)[::-1], new)]
    return new, [k - n for k, n in zip(kv, new)], kv


def _pairs(case):
    """(query, key) pairs that the mask leaves, of one head."""
    n, past, _ = (np.array(x, np.int64) for x in _lengths(case))
    if not case["causal"]:
        return int((n * (past + n)).sum())
    total = int((n * past + n * (n + 1) // 2).sum())
    if case["window"]:
        w = case["window"]
        total = sum(int(np.minimum(np.arange(p + 1, p + k + 1), w).sum()) for p, k in zip(past, n))
    return total


def _keys_read(case):
    new, past, kv = _lengths(case)
    if case["causal"] and case["window"]:
        return sum(min(k, n - 1 + case["window"]) for n, k in zip(new, kv))
    return sum(kv)


def _row_bytes(case):
    """Bytes of one position of one KV head, key or value."""
    D = case["D"]
    return {"bf16": 2 * D, "f32": 4 * D, "int4": D // 2 + D // 32 * 4}[case["kind"]]


def work(case):
    if case["op"] == "rope":
        n = case["T"] * case["heads"] * case["D"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * n * size + case["T"] * (4 + case["rot"] * 4), "flops": case["T"] * case["heads"] * case["rot"] * 3}
    T = sum(_lengths(case)[0])
    size = 4 if case["kind"] == "f32" else 2
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    if case["op"] == "append":
        back = 2 * T * Hkv * D * size if case["kind"] == "int4" else 0
        return {"bytes": T * (2 * H + 2 * Hkv) * D * size + 2 * T * Hkv * _row_bytes(case) + back + T * case["rot"] * 4,
                "flops": T * (H + Hkv) * case["rot"] * 3}
    return {"bytes": 2 * T * H * D * size + 2 * _keys_read(case) * Hkv * _row_bytes(case), "flops": 4 * D * H * _pairs(case)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Angle per position of every pair, and the factor on cosine and sine, for a stretched range of positions."""
    rot, theta = case["rot"], case["theta"]
    kind, f = case.get("scaling", "none"), case.get("factor", 1.0)
    i = torch.arange(rot // 2, dtype=torch.float64)
    if kind == "ntk":
        theta = theta * f ** (rot / (rot - 2))
    w = theta ** (-2.0 * i / rot)
    if kind == "linear":
        return w / f, 1.0
    if kind == "yarn":
        turns = lambda n: rot * math.log(case["orig"] / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(turns(32)), 0), min(math.ceil(turns(1)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _tables(case, n):
    w, m = _frequencies(case)
    a = torch.arange(n, dtype=torch.float64)[:, None] * w[None]
    return (a.cos() * m).float().cuda(), (a.sin() * m).float().cuda()


def _pages(case, kv, g):
    """A table of page numbers in no order, unused entries -1, and how many pages the pool has."""
    ps = case["ps"]
    need = [-(-k // ps) for k in kv]
    n = sum(need) + 3
    order = torch.randperm(n, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    ends = torch.tensor(need, device="cuda").cumsum(0)
    col = torch.arange(max(need), device="cuda")[None]
    idx = (ends - torch.tensor(need, device="cuda"))[:, None] + col
    return torch.where(idx < ends[:, None], order[idx.clamp(max=n - 1)], -1).to(torch.int32), n


def _fill(case, n, g):
    """A cache with content: some key channels are several times as wide as others, as behind a rotation, values are near one."""
    Hkv, D, ps = case["Hkv"], case["D"], case["ps"]
    gain = torch.exp(0.4 * torch.randn(Hkv, 1, D, generator=g, device="cuda"))
    k = torch.randn(n, Hkv, ps, D, generator=g, device="cuda") * gain
    v = torch.randn(n, Hkv, D, ps, generator=g, device="cuda")
    if case["kind"] != "int4":
        return [k.to(_DT[case["kind"]]), v.to(_DT[case["kind"]])]
    kc, km = _quantise(k.unflatten(-1, (D // 32, 32)))
    vc, vm = _quantise(v.transpose(-1, -2).unflatten(-1, (D // 32, 32)))
    return [_pack_k(kc.flatten(-2)), _pack(vc.flatten(-2).transpose(-1, -2)), km.contiguous(), vm.permute(0, 1, 3, 4, 2).contiguous()]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "rope":
        dt = _DT[case["dtype"]]
        s["cos"], s["sin"] = _tables(case, case["max_pos"])
        fused = rnd(case["T"], (case["heads"] + 4) * case["D"]).to(dt)  # rows of a fused projection: other heads lie behind these
        s["x"] = fused[:, : case["heads"] * case["D"]].unflatten(1, (case["heads"], case["D"]))
        s["pos"] = torch.randint(0, case["max_pos"], (case["T"],), generator=g, device="cuda", dtype=torch.int32)
        return s
    new, past, kv = _lengths(case)
    T, dt, H, Hkv, D = sum(new), _DT[case["kind"]], case["H"], case["Hkv"], case["D"]
    s["table"], n = _pages(case, kv, g)
    s["cache"] = _fill(case, n, g)
    s["cu"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["past"], s["kv"] = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in (past, kv))
    s["max_new"], s["max_kv"] = max(new), max(kv)
    if case["op"] == "append":
        s["cos"], s["sin"] = _tables(case, max(kv))
        fused = rnd(T, (H + 2 * Hkv) * D).to(dt)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in fused.split([H * D, Hkv * D, Hkv * D], 1))
    else:
        s["q"] = rnd(T, H, D).to(dt)
    if own:
        from speech_to_speech_amd import paged_kv

        s["handle"] = paged_kv.PagedKVCache.adopt(*s["cache"])
    return s


# ---- the plain form ----------------------------------------------------------------------------------------------------------------


def _turn(x, c, s, rot, inter):
    """x [..., D] in 32 bits turned by the angles whose cosines and sines are given for every pair."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., : rot // 2], x[..., rot // 2 : rot])
    y = torch.stack([a * c - b * s, b * c + a * s], -1 if inter else -2).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _quantise(x):
    """x [..., 32] -> codes 0 .. 15 and (scale, zero) in float16."""
    lo, hi = x.amin(-1), x.amax(-1)
    scale = ((hi - lo) / 15).half()
    zero = (lo + 8 * scale.float()).half()
    s = scale.float()[..., None]
    code = torch.round((x - zero.float()[..., None]) / torch.where(s > 0, s, 1.0)) + 8
    return torch.where(s > 0, code.clamp(0, 15), 8.0).to(torch.uint8), torch.stack([scale, zero], -1)


def _pack(c):
    """Codes [..., 8 n] -> bytes [..., 4 n]: element e of an octet in nibble (e >> 1) + 4 (e & 1)."""
    o = c.unflatten(-1, (-1, 8))[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    return (o[..., :4] | o[..., 4:] << 4).flatten(-2)


def _unpack(b):
    o = b.unflatten(-1, (-1, 4))
    return torch.cat([o & 15, o >> 4], -1)[..., [0, 2, 4, 6, 1, 3, 5, 7]].flatten(-2)


def _pack_k(c):
    n = c.shape[-1] // 32
    return _pack(c.unflatten(-1, (n, 4, 8)).transpose(-2, -3).flatten(-3))


def _unpack_k(b):
    c = _unpack(b)
    return c.unflatten(-1, (4, -1, 8)).transpose(-2, -3).flatten(-3)


def _values(code, meta):
    """Codes and (scale, zero) of groups of 32 -> what they stand for."""
    x = code.unflatten(-1, (-1, 32)).float() - 8
    return (meta[..., 1].float()[..., None] + meta[..., 0].float()[..., None] * x).flatten(-2)


def _rows(s):
    """Session, place among its new rows, position, page and place in the page of every new row."""
    t = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], t, right=True) - 1
    i = t - s["cu"][b]
    p = s["past"][b] + i
    ps = s["case"]["ps"]
    return b, i, p, s["table"][b, p // ps].long(), (p % ps).long()


def _plain_append(s):
    case, rot, inter = s["case"], s["case"]["rot"], s["case"]["inter"]
    b, i, p, page, at = _rows(s)
    c, sn = s["cos"][p][:, None], s["sin"][p][:, None]
    dt = _DT[case["kind"]]
    q = _turn(s["q"].float(), c, sn, rot, inter).to(dt)
    k, v = _turn(s["k"].float(), c, sn, rot, inter).to(dt), s["v"]
    if case["kind"] != "int4":
        s["cache"][0][page, :, at] = k
        s["cache"][1][page, :, :, at] = v
        return {"q": q, "k": s["cache"][0], "v": s["cache"][1]}
    kc, km = _quantise(k.float().unflatten(-1, (-1, 32)))
    vc, vm = _quantise(v.float().unflatten(-1, (-1, 32)))
    ck, cv, mk, mv = s["cache"]
    ck[page, :, at] = _pack_k(kc.flatten(-2))
    mk[page, :, at] = km
    mv[page, :, :, :, at] = vm
    some, where = torch.unique(page, return_inverse=True)  # a byte of values holds two positions: their pages are taken apart and put together
    open_ = _unpack(cv[some])
    open_[where, :, :, at] = vc.flatten(-2)
    cv[some] = _pack(open_)
    return {"q": q, "k": _values(_unpack_k(ck[page, :, at]), mk[page, :, at]).to(dt),
            "v": _values(_unpack(cv[some])[where, :, :, at], mv[page, :, :, :, at]).to(dt)}


def _past(s):
    """Keys and values of all sessions [B][Hkv][S][D] in 32 bits."""
    case, cache = s["case"], s["cache"]
    page = s["table"].clamp(min=0).long()
    put = lambda x: x.transpose(1, 2).flatten(2, 3)  # noqa: E731
    if case["kind"] != "int4":
        return put(cache[0][page].float()), put(cache[1][page].float().transpose(-1, -2))
    k = _values(_unpack_k(cache[0][page]), cache[2][page])
    v = _values(_unpack(cache[1][page]).transpose(-1, -2), cache[3][page].permute(0, 1, 2, 5, 3, 4))
    return put(k), put(v)


def _plain_attend(s):
    case, H, Hkv, D = s["case"], s["case"]["H"], s["case"]["Hkv"], s["case"]["D"]
    k, v = _past(s)
    B, S, n, g = k.shape[0], k.shape[2], s["max_new"], H // Hkv
    t = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], t, right=True) - 1
    i = (t - s["cu"][b]).long()
    q = torch.zeros(B, n, H, D, device="cuda")
    q[b, i] = s["q"].float()
    q = q.unflatten(2, (Hkv, g)).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * n, D)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(B, Hkv, g, n, S)
    key = torch.arange(S, device="cuda")
    last = (s["kv"] - 1)[:, None].expand(B, n)
    if case["causal"]:
        last = s["past"][:, None] + torch.arange(n, device="cuda")
    gone = key > last[..., None]
    if case["window"]:
        gone |= key <= last[..., None] - case["window"]
    gone = gone[:, None, None]
    x = x.masked_fill_(gone, float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True))
    o = torch.matmul(x.view(B, Hkv, g * n, S), v).view(B, Hkv, g, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    return o[b, i].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if own:
        from speech_to_speech_amd import paged_kv

        if case["op"] == "rope":
            return paged_kv.rope(s["x"], s["pos"], s["cos"], s["sin"], interleaved=case["inter"])
        h = s["handle"]
        if case["op"] == "append":
            q = h.append(s["k"], s["v"], s["table"], s["past"], s["cu"], max_new=s["max_new"], cos=s["cos"], sin=s["sin"], interleaved=case["inter"], q=s["q"])
            k, v = h.read(s["table"], s["past"], s["cu"], s["q"].shape[0], max_new=s["max_new"]) if case["kind"] == "int4" else s["cache"]
            return {"q": q, "k": k, "v": v}
        return h.attend(s["q"], s["table"], s["kv"], s["cu"], max_new=s["max_new"], max_kv=s["max_kv"], causal=case["causal"], window=case["window"])
    if case["op"] == "rope":
        p = s["pos"].long()
        x = s["x"]
        return _turn(x.float(), s["cos"][p][:, None], s["sin"][p][:, None], case["rot"], case["inter"]).to(x.dtype)
    return _plain_append(s) if case["op"] == "append" else _plain_attend(s)


# ---- 64 bits, from the definitions -------------------------------------------------------------------------------------------------


def _exact_turn(x, pos, case):
    """Each pair of channels as a complex number times exp(i angle)."""
    rot, f, kind = case["rot"], case.get("factor", 1.0), case.get("scaling", "none")
    half = rot // 2
    base = case["theta"] * (f ** (rot / (rot - 2)) if kind == "ntk" else 1.0)
    w, m = np.array([base ** (-(2 * i) / rot) for i in range(half)]), 1.0
    if kind == "linear":
        w = w / f
    if kind == "yarn":
        bound = [rot / 2 * math.log(case["orig"] / (2 * math.pi * n)) / math.log(base) for n in (32.0, 1.0)]
        lo, hi = max(0, math.floor(bound[0])), min(rot - 1, math.ceil(bound[1]))
        keep = 1 - np.clip((np.arange(half) - lo) / max(hi - lo, 1e-3), 0, 1)
        w, m = w * (keep + (1 - keep) / f), 1 + math.log(f) / 10
    angle = pos.double()[:, None] * torch.from_numpy(w).to(x.device)
    z = torch.polar(torch.full_like(angle, m), angle)[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["inter"] else (slice(0, half), slice(half, rot))
    y = x.double().clone()
    r = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
    y[..., first], y[..., second] = r.real, r.imag
    return y


def _exact_nibbles(rows):
    """What 4 bits hold of rows [..., D] in 64 bits."""
    x = rows.double().reshape(*rows.shape[:-1], -1, 32)
    low = x.min(-1, keepdim=True).values
    step = ((x.max(-1, keepdim=True).values - low) / 15.0).half().double()
    mid = (low + 8 * step).half().double()
    level = ((x - mid) / step.clamp(min=1e-30)).round().clamp(-8, 7)
    return (mid + step * torch.where(step > 0, level, 0.0)).flatten(-2)


def _exact_code(octets):
    """Bytes [..., 4] of an octet -> its 8 codes, from the nibble's place."""
    word = sum(octets[..., j].long() << (8 * j) for j in range(4))
    return torch.stack([(word >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15 for e in range(8)], -1)


def _exact_session(case, cache, pages):
    """Keys and values [Hkv][S][D] of one session, page by page, in 64 bits."""
    D, n = case["D"], case["D"] // 32
    if case["kind"] != "int4":
        return torch.cat([cache[0][p].double() for p in pages], 1), torch.cat([cache[1][p].double().transpose(1, 2) for p in pages], 1)
    keys, values = [], []
    for p in pages:
        dwords = _exact_code(cache[0][p].unflatten(-1, (D // 8, 4)))  # [Hkv][ps][dword][8]
        order = torch.tensor([g * n + s for s in range(n) for g in range(4)], device=dwords.device)
        c = dwords[:, :, order].flatten(-2).double() - 8
        m = cache[2][p].double().repeat_interleave(32, 2)
        keys.append(m[..., 1] + m[..., 0] * c)
        c = _exact_code(cache[1][p].unflatten(-1, (-1, 4))).flatten(-2).double() - 8
        m = cache[3][p].double().repeat_interleave(32, 1)
        values.append((m[:, :, 1] + m[:, :, 0] * c).transpose(1, 2))
    return torch.cat(keys, 1), torch.cat(values, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turn(s["x"], s["pos"], case)
    new, past, kv = _lengths(case)
    D, ps, starts = case["D"], case["ps"], np.concatenate([[0], np.cumsum(new)])
    if case["op"] == "append":
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(past, new)]).cuda()
        q, k, v = _exact_turn(s["q"], pos, case), _exact_turn(s["k"], pos, case), s["v"].double()
        if case["kind"] == "int4":
            return {"q": q, "k": _exact_nibbles(k.to(torch.bfloat16)), "v": _exact_nibbles(v)}
        ks, vs = s["cache"][0].double(), s["cache"][1].double()
        table = s["table"].cpu().numpy()
        for b in range(case["B"]):
            for first in range(past[b] // ps * ps, kv[b], ps):  # one page at a time
                lo, hi = max(first, past[b]), min(first + ps, kv[b])
                page, at, rows = int(table[b, first // ps]), slice(lo - first, hi - first), slice(starts[b] + lo - past[b], starts[b] + hi - past[b])
                ks[page, :, at] = k[rows].transpose(0, 1)
                vs[page, :, :, at] = v[rows].permute(1, 2, 0)
        return {"q": q, "k": ks, "v": vs}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    table = s["table"].cpu().numpy()
    for b in range(case["B"]):
        k, v = _exact_session(case, s["cache"], [int(p) for p in table[b, : -(-kv[b] // ps)]])
        k, v = k[:, : kv[b]], v[:, : kv[b]]
        rows = slice(int(starts[b]), int(starts[b + 1]))
        q = s["q"][rows].double().unflatten(1, (case["Hkv"], -1)).permute(1, 0, 2, 3)  # [Hkv][new][heads][D]
        x = torch.matmul(q.flatten(1, 2), k.transpose(1, 2).contiguous()).unflatten(1, (new[b], -1)) / math.sqrt(D)
        query = past[b] + torch.arange(new[b], device="cuda")[:, None]
        key = torch.arange(kv[b], device="cuda")[None]
        seen = (key <= query) if case["causal"] else torch.ones(new[b], kv[b], dtype=torch.bool, device="cuda")
        if case["window"]:
            seen = seen & (key > query - case["window"])
        x = x.masked_fill(~seen[None, :, None], -math.inf)
        p = torch.softmax(x, -1)
        out[rows] = torch.matmul(p.flatten(1, 2), v).unflatten(1, (new[b], -1)).permute(1, 0, 2, 3).flatten(1, 2)
    return out
