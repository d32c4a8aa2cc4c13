"""The operators that verify drafted tokens, without a GPU: what their entry points refuse before
anything is queued, rows of different lengths that share memory, frequencies."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

from defer_amd import gpu as G
from defer_amd import q8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address that is aligned; nothing reads it on the host
FAR = 1 << 30


def call(name, *args):
    return getattr(q8._lib(), "defer_gpu_q8_" + name)(*args)


def refused(name, *args):
    assert call(name, *args) == G.E_INVALID, (name, args)
    return G.lib().defer_gpu_last_error().decode()


def _cache(**kw):
    d = dict(keys=P, values=P, key_scale=P, value_scale=P, table=P, pages=4, heads=2, head_dim=64, table_width=2)
    d.update(kw)
    return q8._CPages(*[d[n] for n, _ in q8._CPages._fields_])


def _rows(**kw):
    d = dict(row_start=P, kv_len=P, sequences=2, rows=5, most_rows=3)
    d.update(kw)
    return q8._CRows(*[d[n] for n, _ in q8._CRows._fields_])


def _rotary(**kw):
    d = dict(freq=P, position=P, q_norm=P, k_norm=P, eps=1e-6, factor=1.0, rotated=64, interleaved=0)
    d.update(kw)
    return q8._CRotary(*[d[n] for n, _ in q8._CRotary._fields_])


BAD_PAGES = [dict(head_dim=0), dict(head_dim=257), dict(heads=0), dict(heads=65536), dict(keys=None), dict(values=P + 4),
             dict(key_scale=None), dict(value_scale=P + 8), dict(table=None), dict(table_width=1 << 26)]
BAD_ROWS = [dict(kv_len=None), dict(row_start=None), dict(most_rows=6), dict(sequences=1 << 30)]
APPEND = [0, _rotary(), P, 256, 4, P, 128, P, 128, FAR, 256, 0, None]
TREE = [0, P, 256, 4, P, 128, 1.0, None, 0, 0, P, 256, 1, P, 1 << 20, None]


@pytest.mark.parametrize("pages,rows", [(b, {}) for b in BAD_PAGES] + [({}, b) for b in BAD_ROWS])
def test_pages_and_rows_are_refused(pages, rows):
    p, r = _cache(**pages), _rows(**rows)
    refused("kv_append", p, r, *APPEND)
    refused("tree_attention", p, r, *TREE)
    refused("kv_keep", p, r, P, P, FAR, None)


def test_append_refuses():
    p, r = _cache(), _rows()
    for i, bad in ((0, 3), (1, None), (2, None), (2, P + 2), (3, 255), (4, 0), (4, 3), (4, 1 << 17), (5, None), (5, P + 1),
                   (6, 127), (7, None), (8, 127), (9, None), (9, FAR + 2), (10, 255)):
        refused("kv_append", p, r, *[bad if j == i else a for j, a in enumerate(APPEND)])
    for bad in (dict(rotated=63), dict(rotated=66), dict(freq=None), dict(freq=P + 4), dict(position=P + 2), dict(q_norm=P + 2),
                dict(k_norm=P + 3), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(factor=math.nan), dict(factor=math.inf)):
        refused("kv_append", p, r, 0, _rotary(**bad), *APPEND[2:])
    # out lies over q shifted, over k, over v
    for name, q, k, v, out in (("q", P, FAR, FAR, P + 4), ("k", P, FAR + 256 * 3, P, FAR), ("v", P, P, FAR + 256 * 3, FAR)):
        assert f"out overlaps {name}" in refused("kv_append", p, r, 0, _rotary(), q, 256, 4, k, 128, v, 128, out, 256, 0, None)
    none = _rows(sequences=0, rows=0, most_rows=0, row_start=None, kv_len=None)
    assert call("kv_append", p, none, 0, _rotary(), None, 256, 4, None, 128, None, 128, None, 256, 0, None) == G.OK
    assert call("kv_append", p, none, 0, _rotary(rotated=0, freq=None), None, 256, 4, None, 128, None, 128, None, 256, 0, None) == G.OK
    p, r = _cache(heads=64), _rows(rows=(1 << 22) - 1, most_rows=(1 << 22) - 1)
    assert "too many" in refused("kv_append", p, r, 0, _rotary(), P, 4096, 64, P, 4096, P, 4096, 1 << 45, 4096, 0, None)


def test_tree_attention_refuses():
    p, r = _cache(), _rows()
    for i, bad in ((0, 3), (1, None), (2, 255), (3, 0), (3, 3), (3, 1 << 17), (4, None), (4, P + 2), (5, 1 << 31), (10, None),
                   (10, P + 4), (11, 255), (13, P + 8)):
        refused("tree_attention", p, r, *[bad if j == i else a for j, a in enumerate(TREE)])
    assert "at most 64" in refused("tree_attention", p, _rows(rows=100, most_rows=65), *TREE)
    need = call("tree_attention_workspace", p, _rows(), 4, 10000)
    assert need > 0
    long = [10000 if j == 5 else a for j, a in enumerate(TREE)]
    assert "workspace" in refused("tree_attention", p, r, *[need - 1 if j == 14 else a for j, a in enumerate(long)])
    none = _rows(sequences=0, rows=0, most_rows=0, row_start=None, kv_len=None)
    assert call("tree_attention", p, none, 0, None, 256, 4, None, 128, 1.0, None, 0, 0, None, 256, 0, None, 0, None) == G.OK


def test_keep_refuses():
    p, r = _cache(), _rows()
    ok = [P, P, FAR, None]
    for i, bad in ((0, None), (0, P + 2), (1, None), (1, P + 1), (2, None), (2, FAR + 2), (2, P), (2, P + 4), (2, P - 4)):
        refused("kv_keep", p, r, *[bad if j == i else a for j, a in enumerate(ok)])
    assert "at most 64" in refused("kv_keep", p, _rows(rows=100, most_rows=65), *ok)
    assert call("kv_keep", p, _rows(sequences=0, rows=0, most_rows=0, row_start=None, kv_len=None), None, None, None, None) == G.OK


def test_log_probs_refuses():
    ok = [0, P, 100, 4, 100, P, 1.0, 5, P, P, P, P, P, P, 1 << 20, None]
    for i, bad in ((0, 3), (1, None), (1, P + 2), (2, 99), (4, 0), (4, (1 << 20) + 1), (5, P + 2), (6, 0.0), (6, -1.0), (6, math.nan),
                   (6, math.inf), (6, 9e-31), (6, 2e30), (7, 33), (7, 101), (8, None), (9, None), (10, None), (11, None), (12, None),
                   (8, P + 1), (11, P + 2), (13, None), (13, P + 8), (14, 10)):
        refused("log_probs", *[bad if j == i else a for j, a in enumerate(ok)])
    assert "too many" in refused("log_probs", 0, P, 1 << 20, 70000, 1 << 20, None, 1.0, 0, P, P, P, None, None, P, 1 << 40, None)
    assert call("log_probs", 0, None, 100, 0, 100, None, 1.0, 5, None, None, None, None, None, None, 0, None) == G.OK
    assert call("log_probs_workspace", 1 << 30, 100, 5) == 0 and call("log_probs_workspace", 1, 1 << 21, 5) == 0
    one = call("log_probs_workspace", 1, 128256, 20)
    assert one > 0 and call("log_probs_workspace", 2000, 128256, 20) == 2000 * one


def test_python_refuses():
    x = torch.zeros(2, 1, 64)
    pages = q8.Pages(torch.zeros(1, 1, 64, 64, dtype=torch.int8), torch.zeros(1, 1, 64, 64, dtype=torch.int8),
                     torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), torch.zeros(1, 1, dtype=torch.int32))
    n = torch.ones(1, dtype=torch.int32)
    rot = q8.rotary(64, device="cpu")
    for c in (lambda: q8.kv_append(pages, x, x, x, n, rot, n), lambda: q8.tree_attention(x, pages, n, n, n),
              lambda: q8.kv_keep(pages, n, n, n, n), lambda: q8.log_probs(x[0]), lambda: q8.log_probs([1.0])):
        with pytest.raises(ValueError, match="GPU|tensor"):
            c()
    for bad in (None, 3, "x"):
        for c in (lambda: q8.kv_append(pages, bad, x, x, n, rot, n), lambda: q8.tree_attention(bad, pages, n, n, n),
                  lambda: q8.kv_keep(pages, bad, n, n, n), lambda: q8.log_probs(bad)):
            with pytest.raises(ValueError):
                c()
    g = torch.zeros(2, 1, 64, requires_grad=True)
    for c in (lambda: q8.kv_append(pages, g, x, x, n, rot, n), lambda: q8.tree_attention(g, pages, n, n, n), lambda: q8.log_probs(g[0])):
        with pytest.raises(ValueError, match="requires a gradient"):
            c()

    def traced(t):
        q8.log_probs(x[0])
        return t + 1

    with pytest.raises(ValueError, match="trace"):
        torch.jit.trace(traced, torch.zeros(1), check_trace=False)
    for kw in (dict(rotated=3), dict(rotated=-2), dict(rotated=4, theta=0.0), dict(rotated=4, scale=0.0),
               dict(rotated=4, scale=2.0, original_len=0), dict(rotated=4, original_len=10, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            q8.rotary(device="cpu", **kw)
    with pytest.raises(TypeError):
        q8._native().kv_append(1)


def test_frequencies():
    f = q8.rotary(8, 10000.0, device="cpu")
    assert f.freq.dtype == torch.float64 and f.freq.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert q8.rotary(0, device="cpu").freq.shape == (0,)
    assert q8.rotary(8, scale=4.0, device="cpu").freq.tolist() == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-15)
    # 8192 positions: 1304 turns, 130, 13.04, 1.304 of which a tenth lies over one turn towards four
    f = q8.rotary(8, scale=8.0, original_len=8192, device="cpu").freq
    w = (8.192 / (2 * math.pi) - 1) / 3
    assert f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001 * (w + (1 - w) / 8)], rel=1e-14)


def test_overlap_of_rows_of_different_lengths(tmp_path):
    (tmp_path / "probe.cpp").write_text('''
#include "q8_index.h"
extern "C" int share(uint64_t a, int64_t as, uint32_t na, int64_t ar, uint64_t b, int64_t bs, uint32_t nb, int64_t br) {
  return q8::overlap((const void*)a, as, na, ar, (const void*)b, bs, nb, br);
}
''')
    out = str(tmp_path / "libprobe.so")
    subprocess.run(["g++", "-O1", "-Wall", "-shared", "-fPIC", "-I", os.path.join(ROOT, "defer_amd", "csrc"), "-o", out,
                    str(tmp_path / "probe.cpp")], check=True)
    f = ctypes.CDLL(out).share
    u64, i64, u32 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_uint32
    f.argtypes = [u64, i64, u32, i64, u64, i64, u32, i64]
    r = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(20000):
        ar, br = r.randint(1, 6), r.randint(1, 6)
        a_stride, b_stride = ar + r.randint(0, 12), br + r.randint(0, 12)
        if r.random() < 0.5:
            a_stride = b_stride = max(a_stride, b_stride)
        na, nb = r.randint(0, 5), r.randint(0, 5)
        a, b = r.randint(100, 160), r.randint(100, 160)
        rows_a = [range(a + i * a_stride, a + i * a_stride + ar) for i in range(na)]
        rows_b = [range(b + i * b_stride, b + i * b_stride + br) for i in range(nb)]
        shared = bool({x for y in rows_a for x in y} & {x for y in rows_b for x in y})
        want = shared and [list(x) for x in rows_a] != [list(x) for x in rows_b]
        assert f(a, a_stride, na, ar, b, b_stride, nb, br) == want, (a, a_stride, na, ar, b, b_stride, nb, br)
        seen[want] += 1
    assert min(seen.values()) > 2000
