"""GPU: every kernel that the 8-bit product and attention choose between, each
against the formula in 64 bits at sizes that end inside its tiles, and against
its own one-row calls bit by bit.

``product_of`` and ``plan_of`` are the library's rules over again, so that a case
says which kernel it is there for."""
import math

import pytest
import torch

from defer_amd import q8
from test_gpu_q8 import DEV, TYPES, check_linear, fill, i8, i32, make_cache, ref_attention, rnd, starts, values

pytestmark = pytest.mark.gpu


def up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ the product

def product_of(rows, m, k, aligned, near=True):
    def tiles(r, c):
        return up(rows, r) * up(m, c)

    def rounds(n, at_once):
        return up(n, at_once)

    m16 = up(m, 16)
    if rows <= 16:
        return "few 1 1 16" if m16 <= 512 and k >= 2048 else "few 1 1 4"
    if rows <= 64 and (tiles(64, 64) < 192 or not aligned):
        return "few 1 2 8" if m16 * up(rows, 32) <= 256 else "few 2 2 8"
    if not near:
        return "few 2 2 8"
    if not aligned:
        return "few 1 2 8" if tiles(128, 128) < 32 else "tile odd"
    stages = up(k, 128)
    t256 = rounds(tiles(256, 128), 256) * (6.0 + 1.0 * stages)
    t128 = rounds(tiles(128, 128), 256) * (3.0 + 0.7 * stages)
    t64 = rounds(tiles(64, 64), 512) * (2.0 + (0.34 if tiles(64, 64) <= 256 else 0.5) * stages)
    if t256 <= t128 and t256 <= t64:
        return "tile 4 2 3"
    return "tile 2 2 4" if t128 <= t64 else "tile 1 1 4"


# k in every part of the first stages of 128, in 16s where that is what is asked for
PRODUCTS = [("tile 4 2 3", 1023, 8189, k) for k in (16, 112, 128, 144, 256, 272, 400, 528)] + [
    ("tile 2 2 4", 513, 28673, 272), ("tile 4 2 3", 769, 8192, 1040),
    ("tile 2 2 4", 511, 8189, 144), ("tile 2 2 4", 511, 8189, 16), ("tile 2 2 4", 385, 8101, 656), ("tile 4 2 3", 150, 32001, 576),
    ("tile 1 1 4", 64, 16383, 48), ("tile 1 1 4", 301, 577, 1536), ("tile 1 1 4", 65, 1000, 2064),
    ("tile odd", 300, 5000, 1001), ("tile odd", 1001, 1999, 127), ("tile odd", 129, 4097, 129), ("tile odd", 900, 900, 1),
    ("few 2 2 8", 40, 12001, 512), ("few 2 2 8", 33, 9001, 1003), ("few 1 2 8", 63, 999, 77), ("few 1 2 8", 200, 577, 1537),
    ("few 1 1 16", 16, 1001, 2049), ("few 1 1 16", 3, 8177, 4096), ("few 1 1 4", 16, 20001, 333), ("few 1 1 4", 1, 28673, 2064)]


@pytest.mark.parametrize("kernel,rows,m,k", PRODUCTS)
def test_product(kernel, rows, m, k):
    assert product_of(rows, m, k, k % 16 == 0) == kernel
    x, w = i8(rows, k, seed=k), i8(m, k, seed=m)
    g = torch.Generator().manual_seed(1)
    xs, ws = torch.rand(rows, generator=g) * 0.01, torch.rand(m, generator=g) * 0.01
    X, W, XS, WS = (t.to(DEV) for t in (x, w, xs, ws))
    y = q8.linear(X, XS, W, WS)
    check_linear(x, xs, w, ws, torch.float32, y)
    for dtype in TYPES[1:]:  # the same value, rounded once
        assert torch.equal(q8.linear(X, XS, W, WS, dtype=dtype), y.to(dtype))
    for i in sorted({0, 1, rows // 2, max(rows - 2, 0), rows - 1}):
        assert torch.equal(q8.linear(X[i:i + 1], XS[i:i + 1], W, WS), y[i:i + 1]), i


@pytest.mark.parametrize("rows,m,k", [(300, 5000, 1008), (1023, 8189, 256), (130, 9001, 400), (40, 5000, 96), (5, 300, 4096)])
def test_product_of_rows_at_odd_addresses(rows, m, k):
    """Rows of a multiple of 16 codes from odd addresses, or an odd distance apart: the bits of the aligned ones."""
    x, w = i8(rows, k, seed=1).to(DEV), i8(m, k, seed=2).to(DEV)
    g = torch.Generator().manual_seed(1)
    xs, ws = torch.rand(rows, generator=g).to(DEV), torch.rand(m, generator=g).to(DEV)
    want = q8.linear(x, xs, w, ws)
    for pad in (1, 7, 16, 31):
        wide_x, wide_w = torch.zeros(rows, k + pad, dtype=torch.int8, device=DEV), torch.zeros(m, k + pad, dtype=torch.int8, device=DEV)
        wide_x[:, pad:], wide_w[:, pad:] = x, w
        assert torch.equal(q8.linear(wide_x[:, pad:], xs, w, ws), want)
        assert torch.equal(q8.linear(x, xs, wide_w[:, pad:], ws), want)
        assert torch.equal(q8.linear(wide_x[:, pad:], xs, wide_w[:, pad:], ws), want)


@pytest.mark.parametrize("far_x,far_w", [(True, False), (False, True), (True, True)])
def test_product_of_rows_far_apart(far_x, far_w):
    rows, m, k = 70, 50, 608
    x, w = i8(rows, k, seed=1).to(DEV), i8(m, k, seed=2).to(DEV)
    g = torch.Generator().manual_seed(1)
    xs, ws = torch.rand(rows, generator=g).to(DEV), torch.rand(m, generator=g).to(DEV)
    assert product_of(rows, m, k, True, near=False) == "few 2 2 8"

    def spread(t):
        wide = torch.empty(t.shape[0], (1 << 22) + 16, dtype=torch.int8, device=DEV)
        wide[:, :k] = t
        return wide[:, :k]

    assert torch.equal(q8.linear(spread(x) if far_x else x, xs, spread(w) if far_w else w, ws), q8.linear(x, xs, w, ws))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,m,k", [(1023, 8190, 144), (511, 8190, 144), (301, 578, 1536), (300, 5002, 1001)])
def test_product_of_tiles_into_every_layout(rows, m, k, dtype):
    """Stores of two channels a lane, and one by one where rows or addresses are odd: only what is there is written."""
    L = q8._lib()
    x, w = i8(rows, k, seed=1).to(DEV), i8(m, k, seed=2).to(DEV)
    g = torch.Generator().manual_seed(1)
    xs, ws = torch.rand(rows, generator=g).to(DEV), torch.rand(m, generator=g).to(DEV)
    want = q8.linear(x, xs, w, ws, dtype=dtype)
    for stride, at in ((m + 1, 0), (m + 2, 1), (m + 2, 2)):
        y = torch.full((rows * stride + at,), 7.0, dtype=dtype, device=DEV)
        rc = L.defer_gpu_q8_linear(x.data_ptr(), k, xs.data_ptr(), w.data_ptr(), k, ws.data_ptr(), rows, m, k, TYPES.index(dtype),
                                   y[at:].data_ptr(), stride, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        got = y[at:].view(rows, stride)
        assert torch.equal(got[:, :m], want) and (got[:, m:] == 7).all() and (y[:at] == 7).all()


# ------------------------------------------------------------------ attention

def plan_of(seqs, rows, most_rows, nh, nkv, hd, most_len):
    dp = up(hd, 64) * 64
    pairs = most_rows * (nh // nkv)

    def waves_of(r):
        return seqs * nkv * up(pairs, 4 * r)

    if pairs <= 4 or dp > 192:
        r = 1
    elif pairs > 8 and dp == 128 and waves_of(4) >= 2048:
        r = 4
    else:
        r = 2 if pairs <= 8 or waves_of(2) >= 1024 else 1
    units = min(max(up(most_len, 128), 1), 64)
    partials = rows * nh * units * (2 + dp) * 4
    if 1 < units <= 16 and r <= 2 and dp <= 128 and waves_of(r) < 1024:
        mode = "group"
    elif units > 1 and waves_of(r) < 1024 and partials <= 128 << 20:
        mode = "split"
    else:
        mode = "direct"
    return f"{dp // 64} {r} {mode}"


# kernel; sequences' lengths and rows; heads
ATTENTIONS = [
    ("1 1 direct", [128, 64, 1, 77], [1] * 4, 8, 2, 64), ("1 1 group", [1500, 129], [1, 1], 8, 2, 64), ("1 1 split", [3001, 40], [1, 1], 8, 2, 64),
    ("1 1 direct", [100, 64], [100, 64], 32, 2, 64), ("1 2 group", [1500, 129], [1, 1], 8, 1, 64), ("1 2 split", [3001, 40], [1, 1], 8, 1, 64),
    ("1 2 direct", [700], [700], 12, 3, 64), ("1 1 split", [2500], [13], 6, 3, 40),
    ("2 1 direct", [128, 64, 1, 77], [1] * 4, 8, 2, 128), ("2 1 group", [1500, 129], [1, 1], 8, 2, 128), ("2 1 split", [6000, 2100], [1, 1], 32, 8, 128),
    ("2 2 direct", [100, 64], [1, 1], 16, 2, 128), ("2 2 group", [1500, 129], [1, 1], 16, 2, 128), ("2 2 split", [3001, 2049], [1, 2], 8, 2, 128),
    ("2 2 split", [2500], [2], 6, 2, 80), ("2 2 split", [8300], [1], 5, 1, 96), ("2 4 direct", [1100], [1100], 32, 4, 100), ("2 4 direct", [1030], [1030], 32, 4, 128),
    ("3 1 direct", [100, 64], [1, 1], 4, 1, 192), ("3 1 split", [900, 130], [1, 1], 4, 2, 160), ("3 2 direct", [128, 3], [1, 1], 8, 1, 192),
    ("3 2 split", [3001, 129], [1, 1], 8, 1, 192), ("3 2 split", [700], [2], 6, 2, 130), ("3 2 direct", [1030], [1030], 16, 2, 192),
    ("4 1 direct", [100], [1], 6, 2, 256), ("4 1 split", [3001, 300], [1, 1], 6, 2, 256), ("4 1 split", [777], [40], 4, 1, 200), ("4 1 direct", [600], [600], 8, 8, 256),
]


def bound(n, big):
    """How far a head's output may be off, as a norm against that of sum p |v|.

    u = 2^-24 is half a step. A score (exponents of 2, at most `big`) is the result
    of at most 9 roundings of it, each its own: 3 u big of them together, ln 2 of
    that in its probability. The numerator and the denominator are sums of B = n /
    64 + 72 parts at most, with 4 roundings each: 8 B of them, each its own, of a
    root mean square of u / sqrt 3 or less: 4 such deviations, of what a sum that
    grows evenly has (1 / sqrt 3 of the last): 4 / 3 sqrt(8 B) u. Fixed point and
    the quotient: 6 u. (A worst case of all in one direction is sqrt(8 B) times
    as much, and would let a position of 20,000 be left out.)"""
    return 2.0 ** -24 * (2.1 * big + 4 / 3 * math.sqrt(8 * (n / 64 + 72)) + 6)


def near_the_formula(out, q, k, v, pos, hidden, hd):
    want, big, (mass, _) = ref_attention(q, k, v, pos, hidden, hd ** -0.5)
    err = (out.cpu().double() - want).norm(dim=-1)
    limit = bound(len(k), big[..., 0]) * mass.norm(dim=-1)
    assert (err <= limit).all(), float((err / limit.clamp(min=1e-300)).max())


@pytest.mark.parametrize("kernel,lens,counts,nh,nkv,hd", ATTENTIONS)
def test_attention(kernel, lens, counts, nh, nkv, hd):
    assert plan_of(len(lens), sum(counts), max(counts), nh, nkv, hd, max(lens)) == kernel
    pages = make_cache(lens, nkv, hd, seed=3)
    k, v = fill(pages, lens, nkv, hd, seed=4)
    kd, vd = values(k), values(v)
    q = rnd(sum(counts), nh, hd, seed=5)
    h = torch.rand(len(lens), max(lens), generator=torch.Generator().manual_seed(6)) < 0.3
    for hidden in (None, h):
        args = (i32(lens), starts(counts), max(counts), max(lens))
        hid = None if hidden is None else hidden.to(DEV)
        out = q8.attention(q.to(DEV), pages, *args, hidden=hid)
        at = 0
        for i, (n, c) in enumerate(zip(lens, counts)):
            k0 = sum(lens[:i])
            for j in sorted({0, c // 3, c // 2, c - 1}):  # rows all over it
                near_the_formula(out[at + j:at + j + 1], q[at + j:at + j + 1], kd[k0:k0 + n], vd[k0:k0 + n], [n - c + j],
                                 None if hidden is None else hidden[i], hd)
                one = q8.Pages(*pages[:4], pages.table[i:i + 1].contiguous())
                got = q8.attention(q[at + j:at + j + 1].to(DEV), one, i32([n - c + j + 1]), hidden=None if hid is None else hid[i:i + 1])
                assert torch.equal(got, out[at + j:at + j + 1]), (i, j)
            at += c
        for dtype in TYPES[1:]:  # the same value, rounded once
            low = q.to(dtype).to(DEV)
            assert torch.equal(q8.attention(low, pages, *args, hidden=hid), q8.attention(low.float(), pages, *args, hidden=hid).to(dtype))


@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 64), (8, 1, 64), (4, 1, 128), (8, 1, 128), (4, 1, 192), (8, 1, 192), (4, 1, 256)])
@pytest.mark.parametrize("n", [129, 2048, 2049, 8192, 8193, 16384, 16390, 20000])
def test_attention_counts_every_position_once(nh, nkv, hd, n):
    """A value at one position and none at the others: what comes out is its probability."""
    pages = make_cache([n], nkv, hd)
    k, v = fill(pages, [n], nkv, hd, seed=1)
    kd = values(k)
    q = rnd(1, nh, hd, seed=2) * 0.3
    s = torch.einsum("hd,ld->hl", q[0].double(), kd[:, 0]) * hd ** -0.5
    p = torch.softmax(s, 1)
    pages.values.zero_()
    lens = i32([n])
    tight = bound(n, 1.4427 * s.abs().amax())
    for t in sorted({0, 1, 63, 64, 127, 128, 2047, 2048, 8191, 8192, 16383, 16384, n - 2, n - 1}):
        if t >= n:
            continue
        page, at = int(pages.table[0, t // 64]), t % 64
        pages.values[page, 0, :, at] = 100
        pages.value_scale[page, 0, at] = 0.01
        out = q8.attention(q.to(DEV), pages, lens).cpu().double()[0]
        pages.values[page, 0, :, at] = 0
        want = p[:, t:t + 1].expand(-1, hd)
        assert ((out - want).norm(dim=-1) <= (tight + 2.0 ** -22) * want.norm(dim=-1)).all(), t
