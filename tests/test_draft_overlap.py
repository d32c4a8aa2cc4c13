"""What kv_append writes shares no byte with the keys and values it reads: other workgroups
of the launch still read them. The queries' own rows are another matter."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from defer_amd import gpu as G
from defer_amd import q8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address that is aligned; nothing reads it on the host
FAR, FARTHER = 1 << 30, 1 << 31


def append(rows, heads, hd, q, k, v, out, stride):
    pages = q8._CPages(P, P, P, P, P, 4, heads, hd, 2)
    r = q8._CRows(P, P, 1, rows, rows)
    rot = q8._CRotary(P, None, None, None, 1e-6, 1.0, hd // 2 * 2, 0)
    rc = q8._lib().defer_gpu_q8_kv_append(pages, r, 0, rot, q, stride, heads, k, stride, v, stride, out, stride, 0, None)
    return rc, G.lib().defer_gpu_last_error().decode()


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("heads,hd,pad", [(1, 1, 0), (2, 64, 0), (2, 64, 7), (3, 40, 1)])
def test_append_into_the_rows_of_its_keys_or_values_is_refused(rows, heads, hd, pad):
    """As many query heads as the cache has, so that the rows are the same ones throughout."""
    stride = heads * hd + pad
    last = (rows - 1) * stride * 4
    for name, k, v in (("k", FAR, FARTHER), ("v", FARTHER, FAR)):
        for out in (FAR, FAR + last, FAR - last):
            rc, why = append(rows, heads, hd, P, k, v, out, stride)
            assert rc == G.E_INVALID and f"out overlaps {name}" in why, (name, out - FAR, why)


def test_append_over_what_turns_its_rows_is_refused():
    """The norms' weights, positions and frequencies, which every workgroup reads."""
    pages, r = q8._CPages(P, P, P, P, P, 4, 1, 64, 2), q8._CRows(P, P, 1, 3, 3)
    for i, what in ((0, "freq"), (1, "position"), (2, "norm"), (3, "norm")):
        for at in (FAR, FAR + 8, FAR + 2 * 256):
            p = [at if j == i else P for j in range(4)]
            rc = q8._lib().defer_gpu_q8_kv_append(pages, r, 0, q8._CRotary(*p, 1e-6, 1.0, 64, 0), P, 64, 1, P, 64, P, 64, FAR, 64, 0, None)
            why = G.lib().defer_gpu_last_error().decode()
            assert rc == G.E_INVALID and "out overlaps" in why and what in why, (what, why)


def test_rows_that_share_a_byte(tmp_path):
    (tmp_path / "probe.cpp").write_text('''
#include "q8_index.h"
extern "C" int share(uint64_t a, int64_t as, uint32_t na, int64_t ar, uint64_t b, int64_t bs, uint32_t nb, int64_t br) {
  return q8::share((const void*)a, as, na, ar, (const void*)b, bs, nb, br);
}
''')
    out = str(tmp_path / "libprobe.so")
    subprocess.run(["g++", "-O1", "-Wall", "-shared", "-fPIC", "-I", os.path.join(ROOT, "defer_amd", "csrc"), "-o", out,
                    str(tmp_path / "probe.cpp")], check=True)
    f = ctypes.CDLL(out).share
    u64, i64, u32 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_uint32
    f.argtypes = [u64, i64, u32, i64, u64, i64, u32, i64]
    r = random.Random(2)
    seen = {True: 0, False: 0}
    same = 0
    for _ in range(20000):
        ar, br = r.randint(1, 6), r.randint(1, 6)
        a_stride, b_stride = ar + r.randint(0, 12), br + r.randint(0, 12)
        na, nb = r.randint(0, 5), r.randint(0, 5)
        a, b = r.randint(100, 160), r.randint(100, 160)
        if r.random() < 0.2:
            ar, a_stride, na, a = br, b_stride, nb, b
        rows_a = [range(a + i * a_stride, a + i * a_stride + ar) for i in range(na)]
        rows_b = [range(b + i * b_stride, b + i * b_stride + br) for i in range(nb)]
        want = bool({x for y in rows_a for x in y} & {x for y in rows_b for x in y})
        assert f(a, a_stride, na, ar, b, b_stride, nb, br) == want, (a, a_stride, na, ar, b, b_stride, nb, br)
        seen[want] += 1
        same += bool(rows_a) and rows_a == rows_b
    assert min(seen.values()) > 2000 and same > 2000


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (4, 2)])
def test_tensors_that_append_may_not_write(rows, nh, nkv):
    dev, hd = "cuda:0", 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(rows, h, hd, generator=g).to(dev) for h in (nh, nkv, nkv))
    lens, start = torch.tensor([rows], dtype=torch.int32, device=dev), torch.tensor([0, rows], dtype=torch.int32, device=dev)
    rot = q8.rotary(hd, device=dev)

    def pages():
        return q8.new_pages(1, nkv, hd, torch.zeros(1, 1, dtype=torch.int32, device=dev))

    first = pages()
    want = q8.kv_append(first, q, k, v, lens, rot, start, rows)
    before = k.clone(), v.clone()
    if nh == nkv:
        for name, out in (("k", k), ("v", v)):
            untouched = pages()
            kept = [t.clone() for t in untouched]
            with pytest.raises(ValueError, match=f"out overlaps {name}"):
                q8.kv_append(untouched, q, k, v, lens, rot, start, rows, out=out)
            assert all(torch.equal(a, b) for a, b in zip(untouched, kept))
    # beside them in one matrix, and the queries' own rows
    beside = torch.cat([t.flatten(1) for t in (k, v, q)], 1)
    into = beside[:, 2 * nkv * hd:].view(rows, nh, hd)
    kk, vv = beside[:, :nkv * hd].view(rows, nkv, hd), beside[:, nkv * hd:2 * nkv * hd].view(rows, nkv, hd)
    other = pages()
    assert torch.equal(q8.kv_append(other, q, kk, vv, lens, rot, start, rows, out=into), want)
    assert torch.equal(kk, before[0]) and torch.equal(vv, before[1])
    own = pages()
    assert torch.equal(q8.kv_append(own, q, k, v, lens, rot, start, rows, out=q), want) and torch.equal(q, want)
    # (places that were not written hold anything)
    for p in (other, own):
        assert torch.equal(p.keys[:, :, :rows], first.keys[:, :, :rows]) and torch.equal(p.values[..., :rows], first.values[..., :rows])
