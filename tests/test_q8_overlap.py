"""Rows that a call writes and rows that it reads: which of them share memory
(plain arithmetic, against the sets of bytes), and that the 8-bit operators refuse
them unless they are the same rows."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from defer_amd import gpu as G
from defer_amd import q8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # an address that is aligned; nothing reads it on the host


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("q8")
    (d / "probe.cpp").write_text('''
#include "q8_index.h"
extern "C" int share(uint64_t a, int64_t as, uint32_t na, uint64_t b, int64_t bs, uint32_t nb, int64_t row) {
  return q8::overlap((const void*)a, as, na, (const void*)b, bs, nb, row);
}
''')
    out = str(d / "libprobe.so")
    subprocess.run(["g++", "-O1", "-Wall", "-shared", "-fPIC", "-I", os.path.join(ROOT, "defer_amd", "csrc"),
                    "-o", out, str(d / "probe.cpp")], check=True)
    f = ctypes.CDLL(out).share
    u64, i64, u32 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_uint32
    f.argtypes = [u64, i64, u32, u64, i64, u32, i64]
    return f


def test_overlap_is_that_of_the_bytes(overlap):
    r = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(20000):
        row = r.randint(1, 6)
        a_stride, b_stride = row + r.randint(0, 12), row + r.randint(0, 12)
        if r.random() < 0.5:
            b_stride = a_stride
        na, nb = r.randint(0, 5), r.randint(0, 5)
        a, b = r.randint(100, 160), r.randint(100, 160)
        rows_a = [range(a + i * a_stride, a + i * a_stride + row) for i in range(na)]
        rows_b = [range(b + i * b_stride, b + i * b_stride + row) for i in range(nb)]
        shared = bool({x for y in rows_a for x in y} & {x for y in rows_b for x in y})
        want = shared and [list(x) for x in rows_a] != [list(x) for x in rows_b]
        assert overlap(a, a_stride, na, b, b_stride, nb, row) == want, (a, a_stride, na, b, b_stride, nb, row)
        seen[want] += 1
    assert min(seen.values()) > 2000
    # columns of one large matrix, side by side and one byte into each other
    big = 1 << 40
    assert not overlap(big, 1 << 20, 1 << 22, big + 4096, 1 << 20, 1 << 22, 4096)
    assert overlap(big, 1 << 20, 1 << 22, big + 4095, 1 << 20, 1 << 22, 4096)
    assert overlap(big, 1 << 20, 1 << 22, big - 4095, 1 << 20, 1 << 22, 4096)


def refused(name, *args):
    assert getattr(q8._lib(), "defer_gpu_q8_" + name)(*args) == G.E_INVALID, (name, args)
    return G.lib().defer_gpu_last_error().decode()


def test_sum_of_the_norm_that_overlaps_its_inputs_is_refused():
    x, far = 1 << 20, 1 << 24
    for at, what in ((x + 4, "x"), (x - 4, "x"), (x + 5 * 32, "x"), (far + 4, "residual"), (far - 2 * 32, "residual")):
        # 6 rows of 8 floats, one behind the other
        assert what in refused("rms_norm", 0, x, 8, far, 8, P, 1e-5, 6, 8, at, 8, P, P, None)
    assert "x" in refused("rms_norm", 0, x, 16, far, 8, P, 1e-5, 6, 8, x, 8, P, P, None)  # other rows than x's from the second on
    assert "x" in refused("rms_norm", 0, x, 20, far, 8, P, 1e-5, 6, 8, x + 52, 20, P, P, None)  # bytes 52 to 84 of every 80, x has 0 to 32
    assert "weight" in refused("rms_norm", 0, x, 8, far, 8, far << 1, 1e-5, 6, 8, (far << 1) - 32, 8, P, P, None)
    assert "weight" in refused("rms_norm", 0, x, 8, far, 8, far << 1, 1e-5, 1, 8, far << 1, 8, P, P, None)


def test_attention_into_rows_that_overlap_its_queries_is_refused():
    q = 1 << 20
    pages = q8._CPages(P, P, P, P, P, 4, 2, 64, 2)
    rows = q8._CRows(P, P, 2, 5, 3)
    for at, stride in ((q + 16, 256), (q - 16, 256), (q, 512), (q + 2 * 1024, 256)):
        assert "out overlaps q" in refused("attention", pages, rows, 0, q, 256, 4, 128, 1.0, None, 0, 0, at, stride, 0, P, 1 << 20, None)


@pytest.mark.gpu
def test_tensors_that_overlap_are_refused_and_the_same_rows_are_not():
    g = torch.Generator().manual_seed(1)
    buf = torch.randn(40, 64, generator=g).to("cuda:0")
    r, w = torch.randn(20, 64, generator=g).to("cuda:0"), torch.ones(64, device="cuda:0")
    keep = buf.clone()
    for out in (buf[1:21], buf[19:39], buf.view(20, 128)[:, :64]):
        with pytest.raises(ValueError, match="overlaps"):
            q8.rms_norm(buf[:20], w, 1e-5, residual=r, out=out)
        with pytest.raises(ValueError, match="overlaps"):
            q8.rms_norm(r, w, 1e-5, residual=buf[:20], out=out)
    with pytest.raises(G.DeferGpuError, match="weight"):
        q8.rms_norm(buf[:20], buf[25], 1e-5, residual=r, out=buf[20:40])
    assert torch.equal(buf, keep)
    want = q8.rms_norm(buf[:20], w, 1e-5, residual=r)
    got = q8.rms_norm(buf[:20], w, 1e-5, residual=r, out=buf[20:])  # behind it
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    halves = torch.cat([keep[:20], torch.zeros(20, 64, device="cuda:0")], 1)
    got = q8.rms_norm(halves[:, :64], w, 1e-5, residual=r, out=halves[:, 64:])  # beside it
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(halves[:, :64], keep[:20])


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows", [(100, 1), (777, 1), (3000, 1), (300, 300), (1100, 900)])
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (16, 2, 128), (5, 1, 40)])
def test_attention_into_its_queries(n, rows, nh, nkv, hd):
    g = torch.Generator().manual_seed(1)
    dev = "cuda:0"
    pages = q8.new_pages(-(-n // 64), nkv, hd, torch.arange(-(-n // 64), dtype=torch.int32, device=dev)[None])
    k, v, q = (torch.randn(m, h, hd, generator=g).to(dev) for m, h in ((n, nkv), (n, nkv), (rows, nh)))
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    start = [torch.tensor([0, m], dtype=torch.int32, device=dev) for m in (n, rows)]
    q8.kv_write(pages, k, v, lens, start[0], n)
    want = q8.attention(q, pages, lens, start[1], rows, n)
    wide = torch.zeros(rows + 1, nh, hd, device=dev)
    wide[1:] = q
    if rows > 1:
        with pytest.raises(ValueError, match="out overlaps q"):
            q8.attention(wide[1:], pages, lens, start[1], rows, n, out=wide[:-1])
    assert torch.equal(q8.attention(q, pages, lens, start[1], rows, n, out=q), want) and torch.equal(q, want)
