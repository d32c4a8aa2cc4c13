"""The 8-bit operators of include/defer_gpu.h on torch tensors of the GPU.

What a decoder layer needs to run on 8-bit weights, activations and cache: rows
to codes, the norm that leaves codes, the product of codes, the cache in codes
and the attention over it. A row of n values is held as n int8 codes and one
float32 scale (max / 127); the header says what is rounded where.

Every call is queued on torch's current stream of its tensors' device, returns
without waiting and may be captured into a graph. Tensors that the kernels
cannot take as they are (another device, type or layout) are refused with a
ValueError, never copied. Values are float32, bfloat16 or float16.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from .gpu import _check, lib

PAGE = 64
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I8, _I32, _F32, _U8 = torch.int8, torch.int32, torch.float32, torch.uint8


class Pages(NamedTuple):
    """A pool of pages of 64 positions, and the pages of each sequence.

    ``keys`` [pages, heads, 64, D] and ``values`` [pages, heads, D, 64] int8 with
    D the head size rounded up to 64, ``key_scale`` and ``value_scale``
    [pages, heads, 64] float32, ``table`` [sequences, width] int32: positions
    64 j .. 64 j + 63 of sequence i are in page table[i, j]."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor
    table: torch.Tensor


def new_pages(pages: int, heads: int, head_dim: int, table: torch.Tensor) -> Pages:
    """An empty pool on the table's device."""
    d = padded(head_dim)
    dev = table.device
    return Pages(torch.zeros(pages, heads, PAGE, d, dtype=_I8, device=dev),
                 torch.zeros(pages, heads, d, PAGE, dtype=_I8, device=dev),
                 torch.zeros(pages, heads, PAGE, dtype=_F32, device=dev),
                 torch.zeros(pages, heads, PAGE, dtype=_F32, device=dev), table)


def padded(head_dim: int) -> int:
    """The head size as a page holds it."""
    return -(-head_dim // PAGE) * PAGE


class _CPages(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("keys", "values", "key_scale", "value_scale", "table")] + \
               [(n, ctypes.c_uint32) for n in ("pages", "heads", "head_dim", "table_width")]


class _CRows(ctypes.Structure):
    _fields_ = [("row_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p)] + \
               [(n, ctypes.c_uint32) for n in ("sequences", "rows", "most_rows")]


_L = None


def _lib():
    global _L
    if _L is None:
        L = lib()
        u32, i64, f32, sz, vp = (ctypes.c_uint32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t, ctypes.c_void_p)
        pages, rows = ctypes.POINTER(_CPages), ctypes.POINTER(_CRows)
        for name, args, res in (
                ("quantize", [u32, vp, i64, u32, u32, vp, vp, vp], ctypes.c_int),
                ("rms_norm", [u32, vp, i64, vp, i64, vp, f32, u32, u32, vp, i64, vp, vp, vp], ctypes.c_int),
                ("linear", [vp, i64, vp, vp, i64, vp, u32, u32, u32, u32, vp, i64, vp], ctypes.c_int),
                ("kv_write", [pages, rows, u32, vp, i64, vp, i64, vp], ctypes.c_int),
                ("kv_read", [pages, rows, u32, vp, vp, vp], ctypes.c_int),
                ("attention_workspace", [pages, rows, u32, u32], sz),
                ("attention", [pages, rows, u32, vp, i64, u32, u32, f32, vp, i64, u32, vp, i64, vp, sz, vp],
                 ctypes.c_int)):
            f = getattr(L, "defer_gpu_q8_" + name)
            f.argtypes, f.restype = args, res
        _L = L
    return _L


def _need(ok: bool, why: str) -> None:
    if not ok:
        raise ValueError(why)


def _on_gpu(t: torch.Tensor, what: str) -> torch.device:
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{what} is not a tensor on a GPU")
    return t.device


def _take(t, what: str, dev, dtype, shape=None) -> int:
    """The address of a contiguous tensor of this device, type and shape (None: any size)."""
    _need(isinstance(t, torch.Tensor) and t.device == dev and t.dtype == dtype, f"{what}: need {dtype} on {dev}")
    if shape is not None:
        _need(t.dim() == len(shape) and all(b is None or a == b for a, b in zip(t.shape, shape)),
              f"{what}: need shape {tuple(shape)}, got {tuple(t.shape)}")
    _need(t.is_contiguous(), f"{what} is not contiguous")
    return t.data_ptr()


def _row_stride(t, what: str, dev, dtype, shape) -> int:
    """Rows of contiguous values any distance apart: that distance."""
    _need(isinstance(t, torch.Tensor) and t.device == dev and t.dtype == dtype, f"{what}: need {dtype} on {dev}")
    _need(t.dim() == len(shape) and tuple(t.shape) == tuple(shape), f"{what}: need shape {tuple(shape)}, got {tuple(t.shape)}")
    inner = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        _need(size == 1 or stride == inner, f"{what}: the values of a row are not contiguous")
        inner *= size
    if t.shape[0] <= 1:
        return inner
    _need(t.stride(0) >= inner, f"{what}: rows overlap")
    return t.stride(0)


class _Call:
    """The current stream of the tensors' device, which is the current one for the call."""

    __slots__ = ("dev", "prev")

    def __init__(self, dev: torch.device):
        self.dev = dev.index

    def __enter__(self) -> int:
        self.prev = torch._C._cuda_getDevice()
        if self.prev != self.dev:
            torch.cuda.set_device(self.dev)
        return torch._C._cuda_getCurrentRawStream(self.dev)

    def __exit__(self, *a):
        if self.prev != self.dev:
            torch.cuda.set_device(self.prev)


def _type(t: torch.Tensor, what: str) -> int:
    ty = _TYPES.get(t.dtype)
    _need(ty is not None, f"{what}: float32, bfloat16 or float16, not {t.dtype}")
    return ty


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, n] and scales [rows] of x [rows, n]."""
    dev = _on_gpu(x, "x")
    ty = _type(x, "x")
    _need(x.dim() == 2 and x.shape[1] > 0, "x: need [rows, n]")
    st = _row_stride(x, "x", dev, x.dtype, x.shape)
    codes = torch.empty(x.shape, dtype=_I8, device=dev)
    scale = torch.empty(x.shape[0], dtype=_F32, device=dev)
    with _Call(dev) as s:
        _check(_lib().defer_gpu_q8_quantize(ty, x.data_ptr(), st, x.shape[0], x.shape[1], codes.data_ptr(),
                                            scale.data_ptr(), s))
    return codes, scale


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(z, codes, scales): z = x + residual rounded to the type (into ``out``,
    which may be x or residual itself; x where there is no residual), and
    z * weight / sqrt(mean(z^2) + eps) in 8 bits."""
    dev = _on_gpu(x, "x")
    ty = _type(x, "x")
    _need(x.dim() == 2 and x.shape[1] > 0, "x: need [rows, n]")
    rows, n = x.shape
    xs = _row_stride(x, "x", dev, x.dtype, x.shape)
    wp = _take(weight, "weight", dev, x.dtype, (n,))
    rp, rs, zp, zs = None, 0, None, 0
    z = x
    if residual is not None:
        rs = _row_stride(residual, "residual", dev, x.dtype, x.shape)
        rp = residual.data_ptr()
        z = torch.empty((rows, n), dtype=x.dtype, device=dev) if out is None else out
    elif out is not None:
        z = out
    if z is not x or residual is not None:
        zs = _row_stride(z, "out", dev, x.dtype, x.shape)
        zp = z.data_ptr()
    codes = torch.empty((rows, n), dtype=_I8, device=dev)
    scale = torch.empty(rows, dtype=_F32, device=dev)
    with _Call(dev) as s:
        _check(_lib().defer_gpu_q8_rms_norm(ty, x.data_ptr(), xs, rp, rs, wp, eps, rows, n, zp, zs,
                                            codes.data_ptr(), scale.data_ptr(), s))
    return z, codes, scale


def linear(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[rows, m]: x_scale[r] w_scale[m] sum_k x[r, k] w[m, k] of int8 codes x
    [rows, k] and w [m, k], the sum exact."""
    dev = _on_gpu(x, "x")
    ty = _TYPES.get(dtype)
    _need(ty is not None, f"dtype: float32, bfloat16 or float16, not {dtype}")
    _need(x.dim() == 2 and isinstance(w, torch.Tensor) and w.dim() == 2, "need x [rows, k] and w [m, k]")
    rows, k = x.shape
    m = w.shape[0]
    xs = _row_stride(x, "x", dev, _I8, (rows, k))
    ws = _row_stride(w, "w", dev, _I8, (m, k))
    xp, wp = _take(x_scale, "x_scale", dev, _F32, (rows,)), _take(w_scale, "w_scale", dev, _F32, (m,))
    y = torch.empty((rows, m), dtype=dtype, device=dev)
    with _Call(dev) as s:
        _check(_lib().defer_gpu_q8_linear(x.data_ptr(), xs, xp, w.data_ptr(), ws, wp, rows, m, k, ty, y.data_ptr(), m, s))
    return y


def _pages(p: Pages, head_dim: int, dev) -> _CPages:
    _need(isinstance(p.keys, torch.Tensor) and p.keys.dim() == 4, "keys: need [pages, heads, 64, D]")
    n, heads, _, d = p.keys.shape
    _need(1 <= head_dim <= d and d == padded(head_dim), f"head size {head_dim} in pages of {d}")
    return _CPages(_take(p.keys, "keys", dev, _I8, (n, heads, PAGE, d)),
                   _take(p.values, "values", dev, _I8, (n, heads, d, PAGE)),
                   _take(p.key_scale, "key_scale", dev, _F32, (n, heads, PAGE)),
                   _take(p.value_scale, "value_scale", dev, _F32, (n, heads, PAGE)),
                   _take(p.table, "table", dev, _I32, (None, None)), n, heads, head_dim, p.table.shape[1])


def _rows(p: Pages, kv_len, row_start, rows: int, most_rows: int, dev) -> _CRows:
    n = p.table.shape[0]
    _need(0 <= most_rows <= rows, f"most_rows {most_rows} of {rows} rows")
    _need(row_start is not None or rows == n, f"{rows} rows of {n} sequences without row_start")
    return _CRows(None if row_start is None else _take(row_start, "row_start", dev, _I32, (n + 1,)),
                  _take(kv_len, "kv_len", dev, _I32, (n,)), n, rows, most_rows)


def kv_write(pages: Pages, k: torch.Tensor, v: torch.Tensor, kv_len: torch.Tensor,
             row_start: Optional[torch.Tensor] = None, most_rows: Optional[int] = None) -> None:
    """Quantises k and v [rows, heads, head_dim] into the pages: rows row_start[i]
    .. row_start[i + 1] - 1 become the last positions of sequence i, which has
    kv_len[i] with them (without row_start: one row each). No sequence has more
    than most_rows of them (without: all)."""
    dev = _on_gpu(k, "k")
    ty = _type(k, "k")
    _need(k.dim() == 3, "k: need [rows, heads, head_dim]")
    rows, heads, hd = k.shape
    cp = _pages(pages, hd, dev)
    _need(heads == cp.heads, f"k has {heads} heads, the pages {cp.heads}")
    ks, vs = _row_stride(k, "k", dev, k.dtype, k.shape), _row_stride(v, "v", dev, k.dtype, k.shape)
    cr = _rows(pages, kv_len, row_start, rows, (rows if row_start is not None else min(rows, 1)) if most_rows is None else most_rows, dev)
    with _Call(dev) as s:
        _check(_lib().defer_gpu_q8_kv_write(cp, cr, ty, k.data_ptr(), ks, v.data_ptr(), vs, s))


def kv_read(pages: Pages, kv_len: torch.Tensor, row_start: Optional[torch.Tensor], rows: int, head_dim: int,
            most_rows: Optional[int] = None, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [rows, heads, head_dim]: the values of the last positions of each
    sequence, rows given as for kv_write. Rows of no sequence are zeros."""
    dev = _on_gpu(kv_len, "kv_len")
    ty = _TYPES.get(dtype)
    _need(ty is not None, f"dtype: float32, bfloat16 or float16, not {dtype}")
    cp = _pages(pages, head_dim, dev)
    cr = _rows(pages, kv_len, row_start, rows, (rows if row_start is not None else min(rows, 1)) if most_rows is None else most_rows, dev)
    k = torch.empty((rows, cp.heads, head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _Call(dev) as s:
        _check(_lib().defer_gpu_q8_kv_read(cp, cr, ty, k.data_ptr(), v.data_ptr(), s))
    return k, v


def attention(q: torch.Tensor, pages: Pages, kv_len: torch.Tensor, row_start: Optional[torch.Tensor] = None,
              most_rows: Optional[int] = None, most_len: Optional[int] = None, scale: Optional[float] = None,
              hidden: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of q [rows, heads, head_dim] over the pages: each row
    over the positions of its sequence up to its own (rows as for kv_write, which
    has written them), query head h on cache head h // (heads / cache heads).
    ``scale``: 1 / sqrt(head_dim) without. ``hidden`` [sequences, n] uint8 or
    bool: non-zero hides a position. ``most_len``: no sequence is longer
    (without: what the table holds). A row that sees nothing is zeros; rows of
    no sequence are left as ``out`` has them (without ``out``: zeros)."""
    dev = _on_gpu(q, "q")
    ty = _type(q, "q")
    _need(q.dim() == 3, "q: need [rows, heads, head_dim]")
    rows, heads, hd = q.shape
    cp = _pages(pages, hd, dev)
    qs = _row_stride(q, "q", dev, q.dtype, q.shape)
    n = pages.table.shape[0]
    if most_rows is None:
        most_rows = rows if row_start is not None else min(rows, 1)
    cr = _rows(pages, kv_len, row_start, rows, most_rows, dev)
    if most_len is None:
        most_len = PAGE * cp.table_width
    _need(0 <= most_len < 1 << 31, f"most_len {most_len}")
    hp, hs, hn = None, 0, 0
    if hidden is not None:
        _need(isinstance(hidden, torch.Tensor) and hidden.dtype in (_U8, torch.bool) and hidden.dim() == 2,
              "hidden: need [sequences, n] uint8 or bool")
        hs, hn, hp = _row_stride(hidden, "hidden", dev, hidden.dtype, (n, hidden.shape[1])), hidden.shape[1], hidden.data_ptr()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev) if row_start is None else torch.zeros(q.shape, dtype=q.dtype, device=dev)
    os_ = _row_stride(out, "out", dev, q.dtype, q.shape)
    with _Call(dev) as s:
        L = _lib()
        need = L.defer_gpu_q8_attention_workspace(cp, cr, heads, most_len)
        ws = torch.empty(need, dtype=_U8, device=dev) if need else None
        _check(L.defer_gpu_q8_attention(cp, cr, ty, q.data_ptr(), qs, heads, most_len,
                                        hd ** -0.5 if scale is None else scale, hp, hs, hn, out.data_ptr(), os_,
                                        None if ws is None else ws.data_ptr(), need, s))
    return out
