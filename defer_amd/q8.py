"""The 8-bit operators of include/defer_gpu.h on torch tensors of the GPU.

What a decoder layer needs to run on 8-bit weights, activations and cache: rows
to codes, the norm that leaves codes, the product of codes, the cache in codes
and the attention over it. A row of n values is held as n int8 codes and one
float32 scale (max / 127); the header says what is rounded where.

Every call is queued on torch's current stream of its tensors' device, returns
without waiting and may be captured into a graph. Tensors that the kernels
cannot take as they are (another device, type or layout) are refused with a
ValueError, never copied. Values are float32, bfloat16 or float16. There is no
backward: results carry no gradient, and a tensor that requires one is refused
where gradients are on, as is any call under torch.jit.trace.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from .gpu import _check, lib

PAGE = 64


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
    return Pages(torch.zeros(pages, heads, PAGE, d, dtype=torch.int8, device=dev),
                 torch.zeros(pages, heads, d, PAGE, dtype=torch.int8, device=dev),
                 torch.zeros(pages, heads, PAGE, dtype=torch.float32, device=dev),
                 torch.zeros(pages, heads, PAGE, dtype=torch.float32, device=dev), table)


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
    """The C calls, for programs that hold raw device memory."""
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


_N = None


def _native():
    """The calls on tensors (csrc/q8_torch.cpp), bound to the library."""
    global _N
    if _N is None:
        try:
            from . import _q8_torch as native
        except ImportError as e:
            raise ImportError("defer_amd/_q8_torch.so: build it first "
                              f"(python -c 'import __graft_entry__ as g; g.build()'): {e}") from e
        native.bind(lib()._name, torch._C._cuda_getCurrentRawStream, _check, torch.OutOfMemoryError)
        _N = native
    return _N


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, n] and scales [rows] of x [rows, n]."""
    return _native().quantize(x)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(z, codes, scales): z = x + residual rounded to the type (into ``out``,
    which may be x or residual itself, or rows apart from both; x where there is
    no residual), and z * weight / sqrt(mean(z^2) + eps) in 8 bits."""
    return _native().rms_norm(x, weight, eps, residual, out)


def linear(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[rows, m]: x_scale[r] w_scale[m] sum_k x[r, k] w[m, k] of int8 codes x
    [rows, k] and w [m, k], the sum exact."""
    return _native().linear(x, x_scale, w, w_scale, dtype)


def kv_write(pages: Pages, k: torch.Tensor, v: torch.Tensor, kv_len: torch.Tensor,
             row_start: Optional[torch.Tensor] = None, most_rows: Optional[int] = None) -> None:
    """Quantises k and v [rows, heads, head_dim] into the pages: rows row_start[i]
    .. row_start[i + 1] - 1 become the last positions of sequence i, which has
    kv_len[i] with them (without row_start: one row each). No sequence has more
    than most_rows of them (without: all)."""
    _native().kv_write(pages, k, v, kv_len, row_start, most_rows)


def kv_read(pages: Pages, kv_len: torch.Tensor, row_start: Optional[torch.Tensor], rows: int, head_dim: int,
            most_rows: Optional[int] = None, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [rows, heads, head_dim]: the values of the last positions of each
    sequence, rows given as for kv_write. Rows of no sequence are zeros."""
    return _native().kv_read(pages, kv_len, row_start, rows, head_dim, most_rows, dtype)


def attention(q: torch.Tensor, pages: Pages, kv_len: torch.Tensor, row_start: Optional[torch.Tensor] = None,
              most_rows: Optional[int] = None, most_len: Optional[int] = None, scale: Optional[float] = None,
              hidden: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of q [rows, heads, head_dim] over the pages: each row
    over the positions of its sequence up to its own (rows as for kv_write, which
    has written them), query head h on cache head h // (heads / cache heads).
    ``scale``: 1 / sqrt(head_dim) without. ``hidden`` [sequences, n] uint8 or
    bool: non-zero hides a position. ``most_len``: no sequence is longer
    (without: what the table holds). A row that sees nothing is zeros; rows of
    no sequence are left as ``out`` has them (without ``out``: zeros). ``out`` may
    be q itself, or rows apart from it."""
    return _native().attention(q, pages, kv_len, row_start, most_rows, most_len, scale, hidden, out)
