"""The 8-bit operators of include/defer_gpu.h on torch tensors of the GPU.

What a decoder layer needs to run on 8-bit weights, activations and cache: rows
to codes, the norm that leaves codes, the product of codes, the cache in codes
and the attention over it. A row of n values is held as n int8 codes and one
float32 scale (max / 127); the header says what is rounded where.

Every call is queued on torch's current stream of its tensors' device, returns
without waiting and may be captured into a graph. Tensors that the kernels
cannot take as they are (another device, type or layout) are refused with a
ValueError, never copied. Values are float32, bfloat16 or float16. There is no
backward: results carry no gradient.
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
                ("attention", [pages, rows, u32, vp, i64, u32, u32, f32, vp, i64, u32, vp, i64, u32, vp, sz, vp],
                 ctypes.c_int)):
            f = getattr(L, "defer_gpu_q8_" + name)
            f.argtypes, f.restype = args, res
        _L = L
    return _L


def _need(ok: bool, why: str) -> None:
    if not ok:
        raise ValueError(why)


def _gpu_of(t: torch.Tensor, what: str) -> int:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} is not a tensor on a GPU")
    return t.get_device()


def _take(t, what: str, dev: int, dtype, shape) -> int:
    """The address of a contiguous tensor of this device, type and shape."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.shape == shape
            and t.is_contiguous()):
        raise ValueError(f"{what}: need a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{dev}, got " +
                         (f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(type(t))))
    return t.data_ptr()


def _row_stride(t, what: str, dev: int, dtype, shape) -> int:
    """Rows of contiguous values any distance apart: that distance."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev and t.shape == shape):
        raise ValueError(f"{what}: need a {dtype} tensor of shape {tuple(shape)} on cuda:{dev}, got " +
                         (f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(type(t))))
    n = 1
    for size in shape[1:]:
        n *= size
    if t.is_contiguous():
        return n
    inner = 1
    for size, stride in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
        _need(size == 1 or stride == inner, f"{what}: the values of a row are not contiguous")
        inner *= size
    if shape[0] <= 1:
        return n
    _need(t.stride(0) >= n, f"{what}: rows overlap")
    return t.stride(0)


_get_device, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(dev: int, f, *args) -> None:
    """f(*args, current stream of the tensors' device), that device being the current one meanwhile."""
    now = _get_device()
    if now == dev:
        rc = f(*args, _stream_of(dev))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, _stream_of(dev))
    if rc:
        _check(rc)


def _type(t: torch.Tensor, what: str) -> int:
    ty = _TYPES.get(t.dtype)
    if ty is None:
        raise ValueError(f"{what}: float32, bfloat16 or float16, not {t.dtype}")
    return ty


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, n] and scales [rows] of x [rows, n]."""
    dev = _gpu_of(x, "x")
    ty = _type(x, "x")
    _need(x.dim() == 2 and x.shape[1] > 0, "x: need [rows, n]")
    rows, n = x.shape
    st = _row_stride(x, "x", dev, x.dtype, x.shape)
    codes, scale = x.new_empty((rows, n), dtype=_I8), x.new_empty(rows, dtype=_F32)
    _call(dev, _lib().defer_gpu_q8_quantize, ty, x.data_ptr(), st, rows, n, codes.data_ptr(), scale.data_ptr())
    return codes, scale


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(z, codes, scales): z = x + residual rounded to the type (into ``out``,
    which may be x or residual itself; x where there is no residual), and
    z * weight / sqrt(mean(z^2) + eps) in 8 bits."""
    dev = _gpu_of(x, "x")
    ty = _type(x, "x")
    _need(x.dim() == 2 and x.shape[1] > 0, "x: need [rows, n]")
    shape, dtype = x.shape, x.dtype
    rows, n = shape
    xs = _row_stride(x, "x", dev, dtype, shape)
    wp = _take(weight, "weight", dev, dtype, (n,))
    rp, rs, zp, zs = None, 0, None, 0
    z = x if out is None else out
    if residual is not None:
        rs = _row_stride(residual, "residual", dev, dtype, shape)
        rp = residual.data_ptr()
        if out is None:
            z = x.new_empty((rows, n))
            zp, zs = z.data_ptr(), n
    if out is not None:
        zs = _row_stride(z, "out", dev, dtype, shape)
        zp = z.data_ptr()
    codes, scale = x.new_empty((rows, n), dtype=_I8), x.new_empty(rows, dtype=_F32)
    _call(dev, _lib().defer_gpu_q8_rms_norm, ty, x.data_ptr(), xs, rp, rs, wp, eps, rows, n, zp, zs,
          codes.data_ptr(), scale.data_ptr())
    return z, codes, scale


def linear(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[rows, m]: x_scale[r] w_scale[m] sum_k x[r, k] w[m, k] of int8 codes x
    [rows, k] and w [m, k], the sum exact."""
    dev = _gpu_of(x, "x")
    ty = _TYPES.get(dtype)
    _need(ty is not None, f"dtype: float32, bfloat16 or float16, not {dtype}")
    _need(x.dim() == 2 and isinstance(w, torch.Tensor) and w.dim() == 2, "need x [rows, k] and w [m, k]")
    rows, k = x.shape
    m = w.shape[0]
    xs = _row_stride(x, "x", dev, _I8, x.shape)
    ws = _row_stride(w, "w", dev, _I8, (m, k))
    xp, wp = _take(x_scale, "x_scale", dev, _F32, (rows,)), _take(w_scale, "w_scale", dev, _F32, (m,))
    y = x_scale.new_empty((rows, m), dtype=dtype)
    _call(dev, _lib().defer_gpu_q8_linear, x.data_ptr(), xs, xp, w.data_ptr(), ws, wp, rows, m, k, ty, y.data_ptr(), m)
    return y


def _pages(p: Pages, head_dim: int, dev: int) -> _CPages:
    keys, values, key_scale, value_scale, table = p
    _need(isinstance(keys, torch.Tensor) and keys.dim() == 4, "keys: need [pages, heads, 64, D]")
    _need(isinstance(table, torch.Tensor) and table.dim() == 2, "table: need [sequences, width]")
    n, heads, _, d = keys.shape
    if not (1 <= head_dim <= d and d == padded(head_dim)):
        raise ValueError(f"head size {head_dim} in pages of {d}")
    return _CPages(_take(keys, "keys", dev, _I8, (n, heads, PAGE, d)), _take(values, "values", dev, _I8, (n, heads, d, PAGE)),
                   _take(key_scale, "key_scale", dev, _F32, (n, heads, PAGE)),
                   _take(value_scale, "value_scale", dev, _F32, (n, heads, PAGE)),
                   _take(table, "table", dev, _I32, table.shape), n, heads, head_dim, table.shape[1])


def _rows(p: Pages, kv_len, row_start, rows: int, most_rows: Optional[int], dev: int) -> _CRows:
    n = p.table.shape[0]
    if most_rows is None:
        most_rows = rows if row_start is not None else min(rows, 1)
    if not 0 <= most_rows <= rows:
        raise ValueError(f"most_rows {most_rows} of {rows} rows")
    start = None
    if row_start is not None:
        start = _take(row_start, "row_start", dev, _I32, (n + 1,))
    elif rows != n:
        raise ValueError(f"{rows} rows of {n} sequences without row_start")
    return _CRows(start, _take(kv_len, "kv_len", dev, _I32, (n,)), n, rows, most_rows)


def kv_write(pages: Pages, k: torch.Tensor, v: torch.Tensor, kv_len: torch.Tensor,
             row_start: Optional[torch.Tensor] = None, most_rows: Optional[int] = None) -> None:
    """Quantises k and v [rows, heads, head_dim] into the pages: rows row_start[i]
    .. row_start[i + 1] - 1 become the last positions of sequence i, which has
    kv_len[i] with them (without row_start: one row each). No sequence has more
    than most_rows of them (without: all)."""
    dev = _gpu_of(k, "k")
    ty = _type(k, "k")
    _need(k.dim() == 3, "k: need [rows, heads, head_dim]")
    rows, heads, hd = k.shape
    cp = _pages(pages, hd, dev)
    if heads != cp.heads:
        raise ValueError(f"k has {heads} heads, the pages {cp.heads}")
    ks, vs = _row_stride(k, "k", dev, k.dtype, k.shape), _row_stride(v, "v", dev, k.dtype, k.shape)
    cr = _rows(pages, kv_len, row_start, rows, most_rows, dev)
    _call(dev, _lib().defer_gpu_q8_kv_write, cp, cr, ty, k.data_ptr(), ks, v.data_ptr(), vs)


def kv_read(pages: Pages, kv_len: torch.Tensor, row_start: Optional[torch.Tensor], rows: int, head_dim: int,
            most_rows: Optional[int] = None, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [rows, heads, head_dim]: the values of the last positions of each
    sequence, rows given as for kv_write. Rows of no sequence are zeros."""
    dev = _gpu_of(kv_len, "kv_len")
    ty = _TYPES.get(dtype)
    _need(ty is not None, f"dtype: float32, bfloat16 or float16, not {dtype}")
    cp = _pages(pages, head_dim, dev)
    cr = _rows(pages, kv_len, row_start, rows, most_rows, dev)
    k = kv_len.new_empty((rows, cp.heads, head_dim), dtype=dtype)
    v = torch.empty_like(k)
    _call(dev, _lib().defer_gpu_q8_kv_read, cp, cr, ty, k.data_ptr(), v.data_ptr())
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
    dev = _gpu_of(q, "q")
    ty = _type(q, "q")
    _need(q.dim() == 3, "q: need [rows, heads, head_dim]")
    shape, dtype = q.shape, q.dtype
    rows, heads, hd = shape
    cp = _pages(pages, hd, dev)
    qs = _row_stride(q, "q", dev, dtype, shape)
    cr = _rows(pages, kv_len, row_start, rows, most_rows, dev)
    if most_len is None:
        most_len = min(PAGE * cp.table_width, (1 << 31) - 1)
    if not 0 <= most_len < 1 << 31:
        raise ValueError(f"most_len {most_len}")
    hp, hs, hn = None, 0, 0
    if hidden is not None:
        _need(isinstance(hidden, torch.Tensor) and hidden.dtype in (_U8, torch.bool) and hidden.dim() == 2,
              "hidden: need [sequences, n] uint8 or bool")
        hn = hidden.shape[1]
        hs, hp = _row_stride(hidden, "hidden", dev, hidden.dtype, (pages.table.shape[0], hn)), hidden.data_ptr()
    clear = out is None
    if clear:
        out, os_ = q.new_empty(shape), heads * hd
    else:
        os_ = _row_stride(out, "out", dev, dtype, shape)
    L = _lib()
    need = L.defer_gpu_q8_attention_workspace(cp, cr, heads, most_len)
    ws = q.new_empty(need, dtype=_U8) if need else None
    _call(dev, L.defer_gpu_q8_attention, cp, cr, ty, q.data_ptr(), qs, heads, most_len,
          hd ** -0.5 if scale is None else scale, hp, hs, hn, out.data_ptr(), os_, clear,
          None if ws is None else ws.data_ptr(), need)
    return out
