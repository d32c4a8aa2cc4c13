"""The 8-bit operators without a GPU: where rows, positions and pages are (the
arithmetic the kernels use, built for the host), and what the entry points
refuse before they queue anything."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from defer_amd import gpu as G
from defer_amd import q8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------ indexes

PROBE = r"""
#include "q8_index.h"
using namespace q8;
extern "C" {
void span(const int32_t* start, const int32_t* len, uint32_t i, uint32_t rows, int64_t* out) {
  const Span s = span_of(start, len, i, rows);
  out[0] = s.start; out[1] = s.n; out[2] = s.len; out[3] = s.pos(0);
}
int page(const int32_t* table, uint32_t width, uint32_t pages, int64_t block) { return page_of(table, width, pages, block); }
int ulen(int64_t p) { return unit_len(p); }
int ucount(int64_t p) { return unit_count(p); }
int umost(int64_t n) { return most_units(n); }
uint32_t pad(uint32_t n) { return padded(n); }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("q8")
    (d / "probe.cpp").write_text(PROBE)
    out = str(d / "libprobe.so")
    subprocess.run(["g++", "-O1", "-Wall", "-shared", "-fPIC", "-I", os.path.join(ROOT, "defer_amd", "csrc"),
                    "-o", out, str(d / "probe.cpp")], check=True)
    L = ctypes.CDLL(out)
    for f in (L.ulen, L.ucount, L.umost):
        f.argtypes = [ctypes.c_int64]
    L.page.argtypes = [ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int64]
    return L


def _i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


def test_spans_stay_inside_the_call(index):
    out = (ctypes.c_int64 * 4)()

    def span(start, lens, i, rows):
        index.span(None if start is None else _i32(*start), _i32(*lens), i, rows, out)
        return list(out)

    assert span([0, 3, 3, 8], [3, 9, 5], 0, 8) == [0, 3, 3, 0]
    assert span([0, 3, 3, 8], [3, 9, 5], 1, 8) == [3, 0, 9, 9]
    assert span([0, 3, 3, 8], [3, 9, 4], 2, 8) == [3, 5, 4, -1]  # longer than the sequence: a row before 0
    assert span(None, [7, 1], 1, 2) == [1, 1, 1, 0]
    lowest, highest = -2**31, 2**31 - 1
    for bad in ([lowest, highest], [5, 2], [-3, -1], [90, 95], [highest, lowest], [2, highest]):
        start, n, _, _ = span(bad, [4], 0, 6)
        assert 0 <= start <= 6 and n >= 0 and start + n <= 6, bad
    assert span([0, 2], [lowest], 0, 2)[3] == lowest - 2  # in 64 bits


def test_a_bad_page_is_no_page(index):
    t = _i32(2, -1, 5, 0, -2**31, 2**31 - 1)
    assert [index.page(t, 6, 5, b) for b in range(-1, 8)] == [-1, 2, -1, -1, 0, -1, -1, -1, -1]
    assert index.page(t, 6, 6, 2) == 5
    assert index.page(t, 6, 0, 0) == -1
    assert index.page(t, 6, 5, 2**40) == -1
    assert [index.page(None, 3, 2, b) for b in range(4)] == [0, 1, -1, -1]  # no table: page = block


def test_units_cover_every_position_once(index):
    for p in [0, 1, 127, 128, 8191, 8192, 8193, 16383, 16384, 100000, 2**31 - 1]:
        n, u = index.ucount(p), index.ulen(p)
        assert u % q8.PAGE == 0 and (n - 1) * u <= p < n * u, p
        assert n <= index.umost(p + 1), p
    assert index.ucount(-1) == 0
    # no row of a shorter sequence has more units than the call's bound
    for n in (1, 64, 129, 8192, 8200, 20000):
        most = index.umost(n)
        assert all(index.ucount(p) <= most for p in range(0, n, 61)), n


def test_padding(index):
    assert [index.pad(n) for n in (1, 63, 64, 65, 128, 200, 256)] == [64, 64, 64, 128, 128, 256, 256]
    assert [q8.padded(n) for n in (1, 63, 64, 65, 128, 200, 256)] == [64, 64, 64, 128, 128, 256, 256]


# ------------------------------------------------------------------ refusals

P = 4096  # an address that is aligned; nothing reads it on the host


def refused(name, *args):
    rc = getattr(q8._lib(), "defer_gpu_q8_" + name)(*args)
    assert rc == G.E_INVALID, (name, args)
    return G.lib().defer_gpu_last_error().decode()


def test_quantize_refuses():
    ok = [0, P, 8, 2, 8, P, P, None]
    for i, bad in ((0, 3), (1, None), (1, P + 2), (2, 7), (4, 0), (5, None), (6, None)):
        refused("quantize", *[bad if j == i else a for j, a in enumerate(ok)])
    assert q8._lib().defer_gpu_q8_quantize(0, None, 8, 0, 8, None, None, None) == G.OK  # no rows: nothing to do


def test_rms_norm_refuses():
    ok = [1, P, 8, P, 8, P, 1e-5, 2, 8, P, 8, P, P, None]
    for i, bad in ((0, 9), (1, None), (1, P + 1), (2, 5), (3, P + 1), (4, 5), (5, None), (6, -1.0), (6, float("nan")),
                   (6, float("inf")), (8, 0), (10, 7), (11, None), (12, None)):
        refused("rms_norm", *[bad if j == i else a for j, a in enumerate(ok)])
    assert q8._lib().defer_gpu_q8_rms_norm(1, None, 8, None, 0, P, 1e-5, 0, 8, None, 0, None, None, None) == G.OK


def test_linear_refuses():
    ok = [P, 32, P, P, 32, P, 2, 4, 32, 0, P, 4, None]
    for i, bad in ((0, None), (1, 31), (2, None), (3, None), (4, 31), (5, None), (6, 1 << 23), (7, 0), (8, 0),
                   (8, 131072), (9, 3), (10, None), (10, P + 2), (11, 3)):
        refused("linear", *[bad if j == i else a for j, a in enumerate(ok)])
    assert "exact" in refused("linear", P, 1 << 20, P, P, 1 << 20, P, 2, 4, 131072, 0, P, 4, None)
    assert q8._lib().defer_gpu_q8_linear(None, 32, None, P, 32, P, 0, 4, 32, 0, None, 4, None) == G.OK


def _cache(**kw):
    d = dict(keys=P, values=P, key_scale=P, value_scale=P, table=P, pages=4, heads=2, head_dim=64, table_width=2)
    d.update(kw)
    return q8._CPages(*[d[n] for n, _ in q8._CPages._fields_])


def _rows(**kw):
    d = dict(row_start=P, kv_len=P, sequences=2, rows=5, most_rows=3)
    d.update(kw)
    return q8._CRows(*[d[n] for n, _ in q8._CRows._fields_])


BAD_PAGES = [dict(head_dim=0), dict(head_dim=257), dict(heads=0), dict(heads=65536), dict(keys=None), dict(values=P + 4),
             dict(key_scale=None), dict(value_scale=P + 8), dict(table=None), dict(table_width=1 << 26)]
BAD_ROWS = [dict(kv_len=None), dict(row_start=None), dict(most_rows=6), dict(sequences=1 << 30)]


@pytest.mark.parametrize("pages,rows", [(b, {}) for b in BAD_PAGES] + [({}, b) for b in BAD_ROWS])
def test_cache_and_attention_refuse_pages_and_rows(pages, rows):
    p, r = _cache(**pages), _rows(**rows)
    refused("kv_write", p, r, 0, P, 128, P, 128, None)
    refused("kv_read", p, r, 0, P, P, None)
    refused("attention", p, r, 0, P, 256, 4, 128, 1.0, None, 0, 0, P, 256, 0, P, 1 << 20, None)


def test_cache_and_attention_refuse_arguments():
    p, r = _cache(), _rows()
    for bad in ((3, P, 128, P, 128), (0, None, 128, P, 128), (0, P, 127, P, 128), (0, P, 128, None, 128), (0, P, 128, P + 1, 128)):
        refused("kv_write", p, r, *bad, None)
    refused("kv_read", p, r, 5, P, P, None)
    refused("kv_read", p, r, 5, None, None, None)
    refused("kv_read", p, r, 0, P + 2, P, None)
    ok = [0, P, 256, 4, 128, 1.0, None, 0, 0, P, 256, 1, P, 1 << 20, None]
    for i, bad in ((0, 3), (1, None), (2, 255), (3, 0), (3, 3), (3, 1 << 17), (4, 1 << 31), (9, None), (10, 255), (12, P + 8)):
        refused("attention", p, r, *[bad if j == i else a for j, a in enumerate(ok)])
    refused("attention", p, r, 0, P, 256, 4, 128, 1.0, P, 99, 100, P, 256, 0, P, 1 << 20, None)
    need = q8._lib().defer_gpu_q8_attention_workspace(p, _rows(), 4, 10000)
    assert need > 0
    assert "workspace" in refused("attention", p, r, 0, P, 256, 4, 10000, 1.0, None, 0, 0, P, 256, 0, P, need - 1, None)
    refused("attention", p, r, 0, P, 256, 4, 10000, 1.0, None, 0, 0, P, 256, 0, None, need, None)
    none = _rows(sequences=0, rows=0, most_rows=0, row_start=None, kv_len=None)
    assert q8._lib().defer_gpu_q8_attention(p, none, 0, None, 256, 4, 128, 1.0, None, 0, 0, None, 256, 0, None, 0, None) == G.OK
    assert q8._lib().defer_gpu_q8_kv_write(p, none, 0, None, 128, None, 128, None) == G.OK
    assert q8._lib().defer_gpu_q8_attention_workspace(None, r, 4, 10) == 0


def test_calls_too_large_for_a_launch_are_refused():
    big = 1 << 22
    refused("quantize", 0, P, 8, big, 8, P, P, None)
    refused("rms_norm", 1, P, 8, P, 8, P, 1e-5, big, 8, P, 8, P, P, None)
    refused("linear", P, 32, P, P, 32, P, 2, 1 << 28, 32, 0, P, 1 << 28, None)
    refused("linear", P, 32, P, P, 32, P, 2097121, 4, 32, 0, P, 4, None)
    p, r = _cache(heads=64), _rows(rows=big - 1, most_rows=big - 1)
    refused("kv_write", p, r, 0, P, 64 * 64, P, 64 * 64, None)
    refused("kv_read", p, r, 0, P, P, None)
    refused("attention", p, r, 0, P, 1 << 20, 64, 128, 1.0, None, 0, 0, P, 1 << 20, 0, P, 1 << 20, None)
    p, r = _cache(heads=1), _rows(rows=big - 1, most_rows=big - 1)
    refused("attention", p, r, 0, P, 1 << 22, 65535, 128, 1.0, None, 0, 0, P, 1 << 22, 0, P, 1 << 20, None)


def test_python_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(2, 64)
    c = torch.zeros(2, 64, dtype=torch.int8)
    pages = q8.Pages(torch.zeros(1, 1, 64, 64, dtype=torch.int8), torch.zeros(1, 1, 64, 64, dtype=torch.int8),
                     torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), torch.zeros(1, 1, dtype=torch.int32))
    n = torch.ones(1, dtype=torch.int32)
    for call in (lambda: q8.quantize(x), lambda: q8.rms_norm(x, x[0], 1e-5), lambda: q8.linear(c, x[:, 0], c, x[:, 0]),
                 lambda: q8.kv_write(pages, x[:1, None], x[:1, None], n), lambda: q8.kv_read(pages, n, None, 1, 64),
                 lambda: q8.attention(x[:1, None], pages, n), lambda: q8.quantize([1.0])):
        with pytest.raises(ValueError):
            call()


def test_python_refuses_what_is_no_tensor():
    x, n = torch.zeros(2, 64), torch.ones(1, dtype=torch.int32)
    pages = q8.Pages(*[None] * 5)
    for bad in (None, 3, "x", [1.0], np.zeros((2, 64))):
        for call in (lambda: q8.quantize(bad), lambda: q8.rms_norm(bad, x[0], 1e-5), lambda: q8.linear(bad, x, x, x),
                     lambda: q8.kv_write(pages, bad, x, n), lambda: q8.kv_read(pages, bad, n, 1, 64),
                     lambda: q8.attention(bad, pages, n)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: q8.linear(x, x, x), lambda: q8._native().quantize(), lambda: q8._native().attention(1)):
        with pytest.raises(TypeError):
            call()
    for bad in ("no such library", q8.__file__):
        with pytest.raises(ImportError):
            q8._native().bind(bad, None, None, None)
    with pytest.raises(ValueError):
        q8.quantize(x)  # what was bound stays bound
