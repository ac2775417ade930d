"""Plain implementations of the paged cache's operators for tests/test_paged*.py: rows of sessions as lists, one session at a time, 64 bits unless
the operator's definition rounds."""

import torch


def turn(x, pos, cos, sin, interleaved):
    """Rows [T][heads][D] (any float type) turned to int positions [T]: every product and sum rounded to float32, the result to x's type."""
    rot = 2 * cos.shape[1]
    y = x.float().clone()
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    if interleaved:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., : rot // 2].clone(), y[..., rot // 2 : rot].clone()
        y[..., : rot // 2], y[..., rot // 2 : rot] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


def four_bits(x):
    """Rows [..., D] -> (codes [..., D] int64, scale [..., D / 32], zero [..., D / 32] float32 values of float16)."""
    g = x.float().clamp(-32768, 32768).unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15).half().float()
    zero = (lo + 8 * scale).half().float()
    code = torch.round((g - zero[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None]) + 8
    code = torch.where(scale[..., None] > 0, code.clamp(0, 15), 8.0)
    return code.flatten(-2).long(), scale, zero


def four_bit_values(x):
    """What the 4-bit cache stands for, in float32 (zero + scale * (code - 8): the product is exact, one rounding)."""
    code, scale, zero = four_bits(x)
    return (zero[..., None] + scale[..., None] * (code.unflatten(-1, (-1, 32)).float() - 8)).flatten(-2)


def nibbles(octets):
    """Dwords of 8 codes as int64 [...] -> codes [..., 8]: element e in nibble (e >> 1) + 4 (e & 1)."""
    return torch.stack([octets >> (4 * ((e >> 1) + 4 * (e & 1))) & 15 for e in range(8)], -1)


def dwords(b):
    w = b.long().unflatten(-1, (-1, 4))
    return w[..., 0] | w[..., 1] << 8 | w[..., 2] << 16 | w[..., 3] << 24


def page_key_codes(page):
    """Key codes of one page [Hkv][ps][D / 2] -> [Hkv][ps][D]: dword g (D / 32) + s holds channels 32 s + 8 g ..."""
    c = nibbles(dwords(page))  # [Hkv][ps][D / 8][8]
    n = c.shape[-2] // 4
    out = torch.empty(*c.shape[:-2], 8 * 4 * n, dtype=torch.long)
    for g in range(4):
        for s in range(n):
            out[..., 32 * s + 8 * g : 32 * s + 8 * g + 8] = c[..., g * n + s, :]
    return out


def page_value_codes(page):
    """Value codes of one page [Hkv][D][ps / 2] -> [Hkv][ps][D]."""
    return nibbles(dwords(page)).flatten(-2).transpose(-1, -2)


def attend(q, k, v, n, scale, causal=True, window=0, seen=None):
    """One session: q [n][H][D], k / v [S][Hkv][D], all float64 -> (o [n][H][D], sum of |q_d k_d| scale, largest over the seen positions, [n][H]).
    ``seen`` [S] bool: positions that have a page."""
    S, Hkv, H = k.shape[0], k.shape[1], q.shape[1]
    G = H // Hkv
    key, row = torch.arange(S)[None], torch.arange(n)[:, None]
    ok = torch.ones(n, S, dtype=torch.bool)
    if causal:
        ok &= key <= S - n + row
        if window:
            ok &= key > S - n + row - window
    if seen is not None:
        ok &= seen[None]
    o = torch.zeros_like(q)
    size = torch.zeros(n, H, dtype=torch.float64)
    for h in range(H):
        kk, vv = k[:, h // G], v[:, h // G]
        x = (q[:, h] @ kk.T * scale).masked_fill(~ok, -float("inf"))
        m = x.amax(-1, keepdim=True) if S else x.new_full((n, 1), -float("inf"))
        p = torch.exp(x - torch.where(torch.isinf(m), 0.0, m))
        total = p.sum(-1, keepdim=True)
        o[:, h] = torch.where(total > 0, p @ vv / torch.where(total > 0, total, 1.0), 0.0)
        if S:
            size[:, h] = (q[:, h].abs() @ kk.abs().T * abs(scale)).masked_fill(~ok, 0).amax(-1)
    return o, size
