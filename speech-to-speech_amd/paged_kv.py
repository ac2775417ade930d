"""Rotary positions and the paged key / value cache (operators of ``include/s2s_mi355x.h``).

A serving loop whose sessions differ widely in length keeps their keys and values in PAGES of one pool instead of one ``max_pos``-row slot
per session: a page holds ``page_size`` positions of every KV head, a session owns a row of page numbers.  The cache is held in the model
type or in 4 bits (bf16 models; a scale and a zero per 32 channels of a position: 0.31 of the bf16 bytes)::

    cache = PagedKVCache(n_pages=4096, kv_heads=8, head_dim=128, kind="int4", device="cuda:0")
    cos, sin = rope_tables(128, max_pos=131072, theta=1e6, scaling="yarn", factor=4.0, original=32768, device="cuda:0")
    # prompts: session b's new rows are cu[b] .. cu[b + 1] - 1 of q / k / v, behind the start[b] positions it has
    q = cache.append(k, v, table, start, cu, max_new=longest, cos=cos, sin=sin, q=q)
    o = cache.attend(q, table, kv_len, cu, max_new=longest, max_kv=longest_session)
    # one token per session: no cu
    q = cache.append(k, v, table, kv_len, cos=cos, sin=sin, q=q)
    o = cache.attend(q, table, kv_len + 1, max_kv=longest_session + 1)

Everything is enqueued on torch's current stream of the cache's device and nothing synchronises: ``max_new`` and ``max_kv`` are HOST bounds of
the device-side lengths (a captured graph replays with other lengths below them).  Of a session beyond the bounds the rows and positions
beyond are left out; the others keep their places in the session.  Tensors are containers only; there is no CPU path.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

from . import native

KINDS = {"model": native.S2S_KV_MODEL, "int4": native.S2S_KV_INT4}
GROUP = 32  # channels of a position that share a scale and a zero


def _require(cond, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


# The checks of a call's tensors cost as much as its launch: they are plain comparisons, and a message is put together only to be raised.


def _call(device, name, fn, *args):
    """fn(torch's current stream on ``device``, *args) with that device current (it is: the usual case, where torch's guard would cost as much as the launch)."""
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: the operators run on a GPU only")
    index = device.index
    if index == torch._C._cuda_getDevice():
        status = fn(torch._C._cuda_getCurrentRawStream(index), *args)
    else:
        with torch.cuda.device(device):
            status = fn(torch._C._cuda_getCurrentRawStream(index), *args)
    if status:
        native.check(status, name)


def _ints(t, n, device, what):
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: contiguous int32[{n}] on {device} needed, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _rows(t, heads, dim, dtype, device, what):
    """[rows][heads][dim] whose heads lie next to each other (a slice of a fused projection's rows is fine) -> (rows, heads, row stride)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or t.dtype is not dtype or t.device != device or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: {dtype} [rows][{'heads' if heads is None else heads}][{dim}] on {device} needed, got {t.dtype} {tuple(shape)} on {t.device}")
    rs, hs, ds = t.stride()
    if (ds != 1 or (hs != dim and shape[1] != 1)) and t.numel():
        raise ValueError(f"{what}: the heads of a row must lie next to each other, got strides {(rs, hs, ds)}")
    return shape[0], shape[1], rs


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: int = 0):
    """-> (float64 angle per position of every channel pair, factor on cosine and sine).

    ``scaling``: "none"; "linear" (positions divided by ``factor``); "ntk" (theta x factor^(d / (d - 2)): the slowest pair is stretched by
    ``factor``, the fastest kept); "yarn" (pairs that turn more than 32 times within the ``original`` trained positions are kept, those that
    turn less than once are divided by ``factor``, a ramp in between; attention factor 0.1 ln(factor) + 1)."""
    _require(rotary_dim >= 2 and rotary_dim % 2 == 0, f"rotary_dim {rotary_dim} must be even")
    _require(theta > 1 and factor >= 1, f"theta {theta} and factor {factor} must be above 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        _require(rotary_dim > 2, "ntk scaling needs more than one channel pair")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    freq = theta ** (-2.0 * i / rotary_dim)
    if scaling in ("none", "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    _require(scaling == "yarn", f"unknown scaling {scaling!r}")
    _require(original > 0, "yarn scaling needs the original number of positions")

    def pair_that_turns(times):
        return rotary_dim * math.log(original / (times * 2 * math.pi)) / (2 * math.log(theta))

    lo = max(math.floor(pair_that_turns(32)), 0)
    hi = min(math.ceil(pair_that_turns(1)), rotary_dim - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0


def rope_tables(rotary_dim: int, max_pos: int, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0, original: int = 0, device="cuda"):
    """Cosine and sine tables float32 [max_pos][rotary_dim / 2], computed in float64 (the angles of far positions lose all digits in float32)."""
    freq, m = rope_frequencies(rotary_dim, theta, scaling, factor, original)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * freq[None]
    return (a.cos() * m).float().to(device), (a.sin() * m).float().to(device)


def _tables(cos, sin, device):
    """-> (positions, channels that turn, cos pointer, sin pointer)."""
    if cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 \
            or not cos.is_contiguous() or not sin.is_contiguous() or cos.device != device or sin.device != device:
        raise ValueError(f"cos / sin: contiguous float32 [max_pos][rotary_dim / 2] on {device} needed")
    n, half = cos.shape
    return n, 2 * half, cos.data_ptr(), sin.data_ptr()


def rope(x, positions, cos, sin, *, interleaved: bool = False, out=None):
    """Turn the first ``2 * cos.shape[1]`` channels of every head of ``x`` [rows][heads][dim] to its row's position -> ``out`` (new, or given, or
    ``x`` itself; else they share no memory).  ``positions`` int32 [rows]: a negative one leaves the row of ``out`` as it is, one behind the table gives NaN."""
    device, shape = x.device, x.shape
    if len(shape) != 3 or (x.stride(2) != 1 and x.numel()):
        raise ValueError(f"x: [rows][heads][dim] with neighbouring channels needed, got {tuple(shape)}, strides {x.stride()}")
    _ints(positions, shape[0], device, "positions")
    n, rot, cp, sp = _tables(cos, sin, device)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not x.dtype or out.device != device or (out.stride(2) != 1 and out.numel()):
        raise ValueError(f"out must match x, got {out.dtype} {tuple(out.shape)} on {out.device}")
    xs, os = x.stride(), out.stride()
    _call(device, "s2s_op_rope", native.load().s2s_op_rope, x.data_ptr(), xs[0], xs[1], out.data_ptr(), os[0], os[1], positions.data_ptr(), cp, sp, n, shape[0], shape[1], shape[2],
          rot, 1 if interleaved else 0, native.dtype_code(x.dtype))
    return out


class PagedKVCache:
    """A pool of pages for the keys and values of ONE layer, and the operators on it.  ``k`` / ``v`` (and ``k_meta`` / ``v_meta`` of a 4-bit cache) are
    the tensors themselves, in the layout of ``s2s_paged_kv``."""

    def __init__(self, n_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, kind: str = "model", dtype=torch.bfloat16, device="cuda"):
        _require(kind in KINDS, f"unknown cache kind {kind!r} ({', '.join(KINDS)})")
        e = dict(device=device)
        if kind == "model":
            self._bind(torch.empty(n_pages, kv_heads, page_size, head_dim, dtype=dtype, **e), torch.empty(n_pages, kv_heads, head_dim, page_size, dtype=dtype, **e), None, None)
        else:
            _require(dtype == torch.bfloat16, "a 4-bit cache takes bfloat16 rows")
            g = head_dim // GROUP
            self._bind(torch.empty(n_pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, **e), torch.empty(n_pages, kv_heads, head_dim, page_size // 2, dtype=torch.uint8, **e),
                       torch.empty(n_pages, kv_heads, page_size, g, 2, dtype=torch.float16, **e), torch.empty(n_pages, kv_heads, g, 2, page_size, dtype=torch.float16, **e))

    @classmethod
    def adopt(cls, k, v, k_meta=None, v_meta=None) -> "PagedKVCache":
        """A cache over tensors the caller has (kept by reference): the shapes give pages, heads, sizes and kind."""
        self = cls.__new__(cls)
        self._bind(k, v, k_meta, v_meta)
        return self

    def _bind(self, k, v, k_meta, v_meta) -> None:
        _require(k.dim() == 4 and v.dim() == 4 and k.dtype == v.dtype and k.device == v.device and k.is_contiguous() and v.is_contiguous(),
                 "pages: contiguous 4-d tensors of one type on one device needed")
        _require((k_meta is None) == (v_meta is None), "k_meta and v_meta go together")
        n, h, ps, d = k.shape
        if k_meta is None:
            self.kind, self.dtype = "model", k.dtype
            _require(v.shape == (n, h, d, ps), f"values: {(n, h, d, ps)} needed, got {tuple(v.shape)}")
        else:
            self.kind, self.dtype, d = "int4", torch.bfloat16, 2 * d
            _require(k.dtype == torch.uint8 and v.shape == (n, h, d, ps // 2), "4-bit pages: uint8 [pages][heads][page_size][dim / 2] and [pages][heads][dim][page_size / 2]")
            _require(k_meta.dtype == v_meta.dtype == torch.float16 and k_meta.shape == (n, h, ps, d // GROUP, 2) and v_meta.shape == (n, h, d // GROUP, 2, ps)
                     and k_meta.is_contiguous() and v_meta.is_contiguous() and k_meta.device == v_meta.device == k.device, "k_meta / v_meta do not match the pages")
        self.k, self.v, self.k_meta, self.v_meta = k, v, k_meta, v_meta
        self.n_pages, self.kv_heads, self.page_size, self.head_dim, self.device = n, h, ps, d, k.device
        self._kv = native.PagedKVStruct(native.ptr(k), native.ptr(v), native.ptr(k_meta), native.ptr(v_meta), n, ps, h, d, KINDS[self.kind], native.dtype_code(self.dtype))
        self._ref = C.byref(self._kv)
        self._ws: dict = {}  # workspace bytes by the sizes of a call

    def _sessions(self, table, lens, cu, rows, max_new, what):
        """-> (sessions, pages per session, rows, bound of a session's new rows): no rows where the bound leaves none."""
        if table.dtype is not torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.device != self.device:
            raise ValueError(f"table: contiguous int32 [sessions][pages] on {self.device} needed, got {table.dtype} {tuple(table.shape)} on {table.device}")
        b, cols = table.shape
        _ints(lens, b, self.device, what)
        if cu is None:
            if rows != b or max_new not in (None, 1):
                raise ValueError(f"without cu there is one row per session ({rows} rows, {b} sessions, max_new {max_new})")
            return b, cols, rows, 1
        _ints(cu, b + 1, self.device, "cu")
        if max_new is None or max_new > rows:
            max_new = rows
        elif max_new < 0:
            raise ValueError(f"max_new: a number of rows needed, got {max_new}")
        return (b, cols, rows, max_new) if max_new else (b, cols, 0, 1)

    def append(self, k, v, table, start, cu=None, *, max_new=None, cos=None, sin=None, interleaved: bool = False, q=None, q_out=None):
        """Store every session's new rows behind the ``start`` positions its pages hold, keys turned to their positions (``cos`` / ``sin`` None: as they come).
        ``q`` is turned along -> ``q_out`` (new, or given, or ``q`` itself), which is returned."""
        device, dim, dtype = self.device, self.head_dim, self.dtype
        T, _, k_rs = _rows(k, self.kv_heads, dim, dtype, device, "k")
        Tv, _, v_rs = _rows(v, self.kv_heads, dim, dtype, device, "v")
        b, cols, rows, max_new = self._sessions(table, start, cu, T, max_new, "start")
        n, rot, cp, sp = (0, 0, 0, 0) if cos is None and sin is None else _tables(cos, sin, device)
        Tq, H, q_rs, qp, qo_rs, qop = T, 0, 0, 0, 0, 0
        if q is not None:
            if cos is None:
                raise ValueError("queries are turned: cos / sin needed")
            Tq, H, q_rs = _rows(q, None, dim, dtype, device, "q")
            if q_out is None:
                q_out, qo_rs = torch.empty_like(q, memory_format=torch.contiguous_format), H * dim
            else:
                To, _, qo_rs = _rows(q_out, H, dim, dtype, device, "q_out")
                if To != Tq:
                    raise ValueError(f"q_out: {Tq} rows needed, got {To}")
            qp, qop = q.data_ptr(), q_out.data_ptr()
        if Tv != T or Tq != T:
            raise ValueError(f"k, v and q need the same rows, got {T}, {Tv} and {Tq}")
        _call(device, "s2s_op_kv_append_paged", native.load().s2s_op_kv_append_paged, self._ref, k.data_ptr(), k_rs, v.data_ptr(), v_rs, qp, q_rs, qop, qo_rs, H, table.data_ptr(), cols,
              start.data_ptr(), 0 if cu is None else cu.data_ptr(), b, rows, max_new, cp, sp, n, rot, 1 if interleaved else 0)
        return q_out if H else None

    def read(self, table, start, cu=None, rows=None, *, max_new=None):
        """Positions ``start[b] + i`` of every session, back as rows (keys, values) [rows][kv_heads][head_dim] of the model type: what the cache stands for.
        ``rows`` = cu[-1] where ``cu`` is given.  Rows that are left out (behind cu[-1], beyond ``max_new``) hold anything."""
        if rows is None:
            _require(cu is None, "rows: how many rows cu counts")
            rows = table.shape[0]
        shape = (rows, self.kv_heads, self.head_dim)
        b, cols, rows, max_new = self._sessions(table, start, cu, rows, max_new, "start")
        k, v = torch.empty(shape, dtype=self.dtype, device=self.device), torch.empty(shape, dtype=self.dtype, device=self.device)
        _call(self.device, "s2s_op_kv_read_paged", native.load().s2s_op_kv_read_paged, self._ref, table.data_ptr(), cols, start.data_ptr(), 0 if cu is None else cu.data_ptr(), b, rows,
              max_new, k.data_ptr(), v.data_ptr(), self.kv_heads * self.head_dim)
        return k, v

    def workspace_bytes(self, heads: int, sessions: int, rows: int, *, max_new: int = 1, max_kv: int, causal: bool = True, window: int = 0) -> int:
        """Bytes ``attend`` needs beside its buffers for these sizes."""
        n = native.load().s2s_op_attn_paged_ws(self._ref, heads, sessions, rows, max_new, max_kv, 1 if causal else 0, window)
        if n < 0:
            native.check(int(n), "s2s_op_attn_paged_ws")
        return int(n)

    def attend(self, q, table, kv_len, cu=None, *, max_new=None, max_kv=None, scale=None, causal: bool = True, window: int = 0, out=None, workspace=None):
        """softmax(scale q k^T) v over the first ``kv_len[b]`` positions of every session (the new rows' own among them) -> ``out`` (new, or given).
        ``q`` [rows][heads][head_dim], heads a multiple of ``kv_heads``; ``scale`` (any finite number) None: head_dim ** -0.5.  causal: new row i of n sees the positions
        below kv_len - n + i + 1, ``window`` > 0: the last ``window`` of those.  A row that sees nothing is zero; rows that are left out stay as they
        are in ``out`` and hold anything in a new one.  Keys and values that some row sees are finite.  ``workspace``: uint8 tensor of ``workspace_bytes`` (None: taken
        from torch's allocator; one given to calls on several streams at once would be overwritten)."""
        device, dim = self.device, self.head_dim
        T, H, q_rs = _rows(q, None, dim, self.dtype, device, "q")
        b, cols, rows, max_new = self._sessions(table, kv_len, cu, T, max_new, "kv_len")
        if max_kv is None:
            max_kv = cols * self.page_size
        elif not 0 <= max_kv <= cols * self.page_size:
            raise ValueError(f"max_kv: 0 .. {cols * self.page_size} in {cols} pages of {self.page_size}, got {max_kv}")
        window = min(window, 1 << 30)
        if out is None:
            out, o_rs = torch.empty_like(q, memory_format=torch.contiguous_format), H * dim
        else:
            To, _, o_rs = _rows(out, H, dim, self.dtype, device, "out")
            if To != T:
                raise ValueError(f"out: {T} rows needed, got {To}")
        c = 1 if causal else 0
        if workspace is None:
            sizes = (H, b, rows, max_new, max_kv, c, window)
            need = self._ws.get(sizes)
            if need is None:
                need = self.workspace_bytes(H, b, rows, max_new=max_new, max_kv=max_kv, causal=causal, window=window)
                if len(self._ws) >= 4096:
                    self._ws.clear()
                self._ws[sizes] = need
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
        elif workspace.device != device or not workspace.is_contiguous():
            raise ValueError(f"workspace: contiguous on {device} needed")
        ws, ws_bytes = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
        _call(device, "s2s_op_attn_paged", native.load().s2s_op_attn_paged, self._ref, q.data_ptr(), q_rs, out.data_ptr(), o_rs, H, table.data_ptr(), cols, kv_len.data_ptr(),
              0 if cu is None else cu.data_ptr(), b, rows, max_new, max_kv, dim ** -0.5 if scale is None else scale, c, window, ws, ws_bytes)
        return out
