"""GPU: the 8-bit operators (include/defer_gpu.h, defer_amd.q8) against plain
64-bit implementations on the CPU: types, sizes, strides, ragged rows, masks
that leave nothing, values that are not finite, pages that are not there."""
import math
import sys

import numpy as np
import pytest
import torch

from defer_amd import gpu as G
from defer_amd import q8

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# half a step of a type, relative to the value
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def ref_codes(y):
    """Rows of y (64 bits, CPU) as codes and float32 scales, and how far each quotient is from a half."""
    top = y.abs().amax(-1, keepdim=True)
    scale = (top / 127).float()
    scale = torch.where(top < 2.0 ** -100, torch.zeros_like(scale), scale)
    scale = torch.where(torch.isfinite(y).all(-1, keepdim=True) & torch.isfinite(scale), scale, torch.tensor(math.nan))
    quo = torch.where(scale > 0, y / scale.double(), torch.zeros_like(y))
    return torch.round(quo).to(torch.int8), scale[..., 0], (quo - torch.floor(quo) - 0.5).abs()


def same(a, b):
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


# ------------------------------------------------------------------ rows

ROWS = [(1, 1), (3, 7), (1, 64), (5, 576), (2, 1001), (7, 4096), (3, 5003), (2, 14336), (1, 40000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", ROWS)
def test_quantize(rows, n, dtype):
    x = rnd(rows, n, seed=n, dtype=dtype)
    codes, scale = q8.quantize(x.to(DEV))
    want, want_scale, _ = ref_codes(x.double())
    assert torch.equal(codes.cpu(), want) and torch.equal(scale.cpu(), want_scale)


def test_quantize_ties_strides_and_odd_values():
    # a maximum of 127 * 2^e: scale 2^e, so halves are exact ties and go to the even code
    for e in (-3, 0, 4):
        x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 0.0]]) * 2.0 ** e
        codes, scale = q8.quantize(x.to(DEV))
        assert codes.cpu().tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, 0]] and scale.item() == 2.0 ** e
    # 381 / 127 = 3: 4.5 / 3 is a tie whose reciprocal product is not
    assert q8.quantize(torch.tensor([[381.0, 4.5, 7.5]], device=DEV))[0].cpu().tolist() == [[127, 2, 2]]
    wide = rnd(6, 300, seed=1).to(DEV)
    for view in (wide[:, 3:200], wide[::2, 1:], wide[:1, 5:6]):
        codes, scale = q8.quantize(view)
        want, want_scale, _ = ref_codes(view.cpu().double())
        assert torch.equal(codes.cpu(), want) and torch.equal(scale.cpu(), want_scale)
    x = rnd(6, 100, seed=2)
    x[0] = 0
    x[1] *= 2.0 ** -140
    x[2, 3] = math.inf
    x[3, 99] = math.nan
    x[4] *= 2.0 ** 120
    x[5, :] = torch.finfo(torch.float32).max
    codes, scale = q8.quantize(x.to(DEV))
    want, want_scale, _ = ref_codes(x.double())
    assert torch.equal(codes.cpu(), want) and same(scale, want_scale)
    assert scale[0] == 0 and scale[1] == 0 and torch.isnan(scale[2:4]).all() and not codes[:4].any()
    assert q8.quantize(torch.empty(0, 5, device=DEV))[0].shape == (0, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", ROWS)
def test_rms_norm(rows, n, dtype):
    x, r, w = rnd(rows, n, seed=1, dtype=dtype), rnd(rows, n, seed=2, dtype=dtype, scale=3), 1 + rnd(n, seed=3, dtype=dtype) / 4
    w = w.to(dtype)
    eps = 1e-5
    for res in (r, None):
        z = x if res is None else (x.float() + res.float()).to(dtype)
        d = z.double()
        y = d / torch.sqrt(d.square().mean(1, keepdim=True) + float(np.float32(eps))) * w.double()
        want, want_scale, off = ref_codes(y)
        got, codes, scale = q8.rms_norm(x.to(DEV), w.to(DEV), eps, residual=None if res is None else res.to(DEV))
        assert torch.equal(got.cpu(), z)
        # the scale is rounded once from 64 bits whose last places depend on the sum's order
        assert torch.allclose(scale.cpu(), want_scale, rtol=2.0 ** -23, atol=0)
        # codes differ only where the quotient is a 64-bit rounding from a half
        far = (codes.cpu() != want) & (off > 1e-6)
        assert not far.any() and (codes.cpu().int() - want.int()).abs().max() <= 1
        assert (codes.cpu() != want).sum() <= 1


def test_rms_norm_in_place_strides_and_odd_values():
    x, r, w = rnd(5, 130, seed=1), rnd(5, 130, seed=2), rnd(130, seed=3)
    z0, c0, s0 = q8.rms_norm(x.to(DEV), w.to(DEV), 1e-6, residual=r.to(DEV))
    for into in ("x", "residual", "apart"):
        wide = torch.full((5, 400), 7.0, device=DEV)
        a, b = wide[:, :130], wide[:, 150:280]
        a.copy_(x)
        b.copy_(r)
        out = {"x": a, "residual": b, "apart": wide[:, 270:400] if into == "apart" else None}[into]
        if into == "apart":
            b = r.to(DEV)
        z, c, s = q8.rms_norm(a, w.to(DEV), 1e-6, residual=b, out=out)
        assert z is out and torch.equal(z, z0) and torch.equal(c, c0) and torch.equal(s, s0)
        assert (wide[:, 130:150] == 7).all()
    x = rnd(4, 66, seed=4)
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 65] = math.nan
    z, c, s = q8.rms_norm(x.to(DEV), torch.ones(66, device=DEV), 1e-5)
    assert s[0] == 0 and torch.isnan(s[1:3]).all() and torch.isfinite(s[3]) and not c[:3].any() and c[3].any()
    w = torch.ones(66)
    w[3] = math.nan
    assert torch.isnan(q8.rms_norm(rnd(2, 66).to(DEV), w.to(DEV), 1e-5)[2]).all()
    with pytest.raises(ValueError):
        q8.rms_norm(x.to(DEV), torch.ones(65, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        q8.rms_norm(x.to(DEV).t(), torch.ones(4, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        q8.rms_norm(x.to(DEV), torch.ones(66, device=DEV), 1e-5, residual=x.to(DEV).half())
    with pytest.raises(G.DeferGpuError):
        q8.rms_norm(x.to(DEV), torch.ones(66, device=DEV), -1.0)


def test_a_row_is_the_same_in_every_call():
    for n in (200, 4096, 9000):
        x, r, w = rnd(9, n, seed=1).to(DEV), rnd(9, n, seed=2).to(DEV), rnd(n, seed=3).to(DEV)
        z, c, s = q8.rms_norm(x, w, 1e-5, residual=r)
        for i in (0, 4, 8):
            zi, ci, si = q8.rms_norm(x[i:i + 1], w, 1e-5, residual=r[i:i + 1])
            assert torch.equal(zi, z[i:i + 1]) and torch.equal(ci, c[i:i + 1]) and torch.equal(si, s[i:i + 1])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_is_the_same_at_every_stride_and_alignment(dtype):
    for n in (64, 1000, 4096, 9000, 20000):
        x, r, w = (rnd(*shape, seed=i, dtype=dtype).to(DEV) for i, shape in enumerate([(7, n), (7, n), (n,)]))
        want = q8.rms_norm(x, w, 1e-5, residual=r)
        for pad in (1, 3, 16):  # rows an odd distance apart, from an odd address on
            wide = torch.zeros(7, n + pad, dtype=dtype, device=DEV)
            wide[:, pad:] = x
            odd = torch.zeros(n + 1, dtype=dtype, device=DEV)
            odd[1:] = w
            for weight in (w, odd[1:]):
                assert all(torch.equal(a, b) for a, b in zip(q8.rms_norm(wide[:, pad:], weight, 1e-5, residual=r), want))
            assert all(torch.equal(a, b) for a, b in zip(q8.quantize(wide[:, pad:]), q8.quantize(x)))


# ------------------------------------------------------------------ the product

def i8(*shape, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(-127, 128, shape, dtype=np.int8))


def check_linear(x, xs, w, ws, dtype, y):
    acc = (x.double() @ w.double().t())  # exact: under 2^53
    want = acc * xs.double()[:, None] * ws.double()
    # the sum to f32, the scales' product, the product, the type: half a step each
    tol = (3 * HALF[torch.float32] + HALF[dtype]) * 1.01 * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((y.cpu().double() - want).abs() <= tol).all()


LINEAR = [(1, 1, 1), (1, 16, 64), (1, 960, 576), (2, 17, 15), (3, 100, 1000), (16, 33, 128), (17, 64, 200), (15, 576, 1536),
          (31, 257, 64), (33, 250, 4096), (64, 512, 2048), (65, 300, 130), (100, 129, 257), (128, 256, 512),
          (200, 500, 1024), (301, 576, 1536), (513, 130, 96), (256, 1000, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,m,k", LINEAR)
def test_linear(rows, m, k, dtype):
    x, w = i8(rows, k, seed=k), i8(m, k, seed=m)
    xs, ws = torch.rand(rows) * 0.01, torch.rand(m) * 0.01
    y = q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), dtype=dtype)
    assert y.dtype == dtype
    check_linear(x, xs, w, ws, dtype, y)


@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_linear_largest_sums_are_exact(rows):
    k = 131071
    x = torch.full((rows, k), -128, dtype=torch.int8)
    w = torch.stack([torch.full((k,), 127, dtype=torch.int8), torch.full((k,), -128, dtype=torch.int8)])
    w[0, 77] = 5  # a sum that f32 would not hold
    y = q8.linear(x.to(DEV), torch.ones(rows, device=DEV), w.to(DEV), torch.ones(2, device=DEV))
    want = (x[0].long() * w.long()).sum(1)
    assert y.cpu().long().sub(want).abs().max() <= 64  # half a step of f32 at 2^31


def test_linear_strides_alignment_and_scales():
    big, wig = i8(70, 700, seed=1).to(DEV), i8(90, 700, seed=2).to(DEV)
    xs, ws = torch.rand(70, device=DEV), torch.rand(90, device=DEV)
    for rows in (1, 9, 70):
        for k0, k1 in ((0, 512), (16, 528), (1, 513), (3, 700), (0, 1)):
            x, w = big[:rows, k0:k1], wig[:, k0:k1]
            y = q8.linear(x, xs[:rows], w, ws)
            check_linear(x.cpu(), xs[:rows].cpu(), w.cpu(), ws.cpu(), torch.float32, y)
            # every layout the same bits
            assert torch.equal(y, q8.linear(x.contiguous(), xs[:rows], w.contiguous(), ws))
    xs[2], xs[3], ws[5] = math.nan, 0.0, math.inf
    y = q8.linear(big, xs, wig, ws)
    assert torch.isnan(y[2]).all() and not y[3, :5].any() and torch.isnan(y[3, 5]) and torch.isinf(y[0, 5])
    assert q8.linear(big[:0], xs[:0], wig, ws).shape == (0, 90)
    with pytest.raises(ValueError):
        q8.linear(big, xs, wig[:, :699], ws)
    with pytest.raises(ValueError):
        q8.linear(big, xs[:69], wig, ws)
    with pytest.raises(ValueError):
        q8.linear(big, xs, wig, ws, dtype=torch.int32)


@pytest.mark.parametrize("rows,m", [(1, 40), (33, 100), (130, 200)])
def test_linear_scales_whose_product_is_below_the_type(rows, m):
    x, w = i8(rows, 4096, seed=1), i8(m, 4096, seed=2)
    x[0] = 0
    for a, b in ((2.0 ** -105, 1.3 * 2.0 ** -30), (1.7 * 2.0 ** -30, 2.0 ** -100), (1e20, 1e19)):
        xs, ws = torch.full((rows,), a), torch.full((m,), b)
        y = q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV)).cpu().double()
        assert not y[0].any()
        want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
        # the sum to f32 and two products: half a step each, or half the least number of the type
        far = (y - want).abs() - torch.clamp(3.03 * HALF[torch.float32] * want.abs(), min=2.0 ** -149)
        fits = want.abs() < 3.4e38
        assert (far[fits] <= 0).all() and torch.isinf(y[~fits]).all()


def test_linear_rows_are_the_same_in_every_call():
    for m, k in ((200, 640), (130, 1000)):
        x, w = i8(300, k, seed=1).to(DEV), i8(m, k, seed=2).to(DEV)
        xs, ws = torch.rand(300, device=DEV), torch.rand(m, device=DEV)
        y = q8.linear(x, xs, w, ws)
        for a, b in ((0, 1), (7, 20), (100, 164), (20, 300)):
            assert torch.equal(q8.linear(x[a:b], xs[a:b], w, ws), y[a:b])


# ------------------------------------------------------------------ the cache

def make_cache(lens, heads, hd, seed=0, spare=3, width=None):
    """Empty pages for sequences of these lengths in an order of their own, full of odd values."""
    per = [-(-n // q8.PAGE) for n in lens]
    g = torch.Generator().manual_seed(seed)
    pool = sum(per) + spare
    order = torch.randperm(pool, generator=g).int()
    table = torch.full((len(lens), max(max(per), 1) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += p
    pages = q8.new_pages(pool, heads, hd, table.to(DEV))
    pages.keys.random_(-128, 128)
    pages.values.random_(-128, 128)
    pages.key_scale.fill_(math.nan)
    pages.value_scale.fill_(math.nan)
    return pages


def starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEV)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def fill(pages, lens, heads, hd, seed=0, dtype=torch.float32, scale=1.0):
    """Whole sequences written; the k and v given."""
    k, v = rnd(sum(lens), heads, hd, seed=seed, dtype=dtype, scale=scale), rnd(sum(lens), heads, hd, seed=seed + 1, dtype=dtype)
    q8.kv_write(pages, k.to(DEV), v.to(DEV), i32(lens), starts(lens), max(lens))
    return k, v


def values(x):
    """What codes of x stand for, in 64 bits."""
    c, s, _ = ref_codes(x.double())
    return c.double() * s.double()[..., None]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hd", [(1, 1), (3, 64), (2, 16), (2, 40), (1, 100), (8, 128), (2, 200), (1, 256)])
def test_cache_written_and_read(heads, hd, dtype):
    lens = [1, 63, 64, 65, 130, 7]
    pages = make_cache(lens, heads, hd, seed=hd)
    k, v = fill(pages, lens, heads, hd, dtype=dtype)
    rk, rv = q8.kv_read(pages, i32(lens), starts(lens), sum(lens), hd)
    for got, x in ((rk, k), (rv, v)):
        want = values(x)
        assert ((got.cpu().double() - want).abs() <= HALF[torch.float32] * 1.01 * want.abs()).all()
    # the last rows alone, in the values' type
    back = [1, 5, 64, 2, 70, 7]
    pk, pv = q8.kv_read(pages, i32(lens), starts(back), sum(back), hd, dtype=dtype)
    at = 0
    for i, (n, b) in enumerate(zip(lens, back)):
        end = sum(lens[:i + 1])
        assert torch.equal(pk[at:at + b], rk[end - b:end].to(dtype)) and torch.equal(pv[at:at + b], rv[end - b:end].to(dtype))
        at += b


def test_cache_row_by_row_equals_at_once_and_touches_nothing_else():
    lens, heads, hd = [5, 64, 129, 200], 3, 72
    pages = make_cache(lens, heads, hd, seed=1)
    before = [t.clone() for t in pages]
    k, v = fill(pages, lens, heads, hd, seed=5)
    other = q8.Pages(*[t.clone() for t in before])
    start = np.cumsum([0] + lens)
    for t in range(max(lens)):  # a row for each sequence that has one left; the others give none
        live = [i for i, n in enumerate(lens) if t < n]
        rows = [int(start[i]) + t for i in live]
        counts = [1 if i in live else 0 for i in range(len(lens))]
        q8.kv_write(other, k[rows].to(DEV), v[rows].to(DEV), i32([min(t + 1, n) for n in lens]), starts(counts), 1)
    for a, b in zip(pages, other):
        assert same(a, b)
    written = torch.zeros(before[0].shape[:1] + (q8.PAGE,), dtype=torch.bool)
    table = pages.table.cpu()
    for i, n in enumerate(lens):
        for t in range(n):
            written[table[i, t // 64], t % 64] = True
    w = written[:, None].expand(-1, heads, -1)
    assert torch.equal(torch.isnan(pages.key_scale.cpu()), ~w) and torch.equal(torch.isnan(pages.value_scale.cpu()), ~w)
    assert torch.equal(pages.keys.cpu()[~w], before[0].cpu()[~w])
    assert torch.equal(pages.values.cpu().transpose(2, 3)[~w], before[1].cpu().transpose(2, 3)[~w])


def test_cache_rows_of_no_sequence_bad_pages_and_odd_values():
    lens, heads, hd = [70, 66], 2, 64
    pages = make_cache(lens, heads, hd)
    table = pages.table.clone()
    table[0, 1] = 1000  # past the pool
    table[1, 0] = -5
    pages = pages._replace(table=table)
    before = [t.clone() for t in pages]
    k, v = rnd(140, heads, hd, seed=1), rnd(140, heads, hd, seed=2)
    k[3, 0, 5], v[4, 1, 7], k[5, 1] = math.inf, math.nan, 0
    args = (i32(lens), i32([1, 71, 137]))  # row 0 and the last three are nobody's
    q8.kv_write(pages, k.to(DEV), v.to(DEV), *args, most_rows=70)
    rk, rv = q8.kv_read(pages, *args, rows=140, head_dim=hd, most_rows=70)
    have = torch.zeros(140, dtype=torch.bool)
    have[1:65] = True     # the first page of sequence 0
    have[135:137] = True  # the second of sequence 1
    for got, x in ((rk, k), (rv, v)):
        want = values(x)
        want[~have] = 0
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert ((got - want).nan_to_num().abs() <= 1e-7 * want.nan_to_num().abs()).all()
    assert torch.isnan(rk[3, 0]).all() and not torch.isnan(rk[3, 1]).any() and not rk[5, 1].any()
    used = {int(table[0, 0]), int(table[1, 1])}
    for p in range(len(before[0])):
        if p not in used:
            assert all(same(a[p], b[p]) for a, b in zip(pages[:4], before[:4]))
    # more rows than the sequence has positions: the first ones are before position 0
    fresh = make_cache([4], heads, hd)
    q8.kv_write(fresh, k[:6].to(DEV), v[:6].to(DEV), i32([4]), i32([0, 6]), 6)
    rk, _ = q8.kv_read(fresh, i32([4]), i32([0, 6]), 6, hd)
    want = values(k[:6])
    want[:2] = 0
    assert torch.equal(torch.isnan(rk.cpu()), torch.isnan(want))
    assert ((rk.cpu().double() - want).nan_to_num().abs() <= 1e-7 * want.nan_to_num().abs()).all()


# ------------------------------------------------------------------ attention

def ref_attention(q, k, v, pos, hidden, scale):
    """q [n, nh, hd] at positions pos of one sequence, k and v [len, nkv, hd], 64
    bits: the output, the largest score (in exponents of 2) and sum p |v|."""
    n, nh, hd = q.shape
    g = nh // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("nhd,lhd->nhl", q.double(), kk) * scale
    off = torch.arange(len(k))[None, :] > torch.as_tensor(pos)[:, None]
    if hidden is not None:
        m = min(len(hidden), len(k))
        off[:, :m] |= hidden[:m].bool()[None]
    s = s.masked_fill(off[:, None], -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(off[:, None].expand_as(p), torch.zeros_like(p), p)
    vz = torch.where((~off).any(0)[:, None, None], vv, torch.zeros_like(vv))
    out = torch.einsum("nhl,lhd->nhd", p, vz)
    nothing = off.all(1)
    out[nothing] = 0
    big = s.masked_fill(off[:, None], 0).abs().amax(-1, keepdim=True) * 1.4427
    top = vz.abs().nan_to_num().amax((0, 2))[None, :, None] if len(vz) else 0.0
    return out, big, (torch.einsum("nhl,lhd->nhd", p.nan_to_num(), vz.abs().nan_to_num()), top)


def tolerance(dtype, length, big, mass, want):
    """An output's error in f32 arithmetic, u = 2^-24 half a step.

    Scores, in exponents of 2, at most `big`: two roundings of the digit sums, one
    joining them, three in the scales (q's are powers of two; scale * log2(e)
    once, its constant once, times the key's scale, times the sum), so at most 7 u
    big; subtracting the block's maximum: 2 u big. A probability is off by ln 2 *
    9 u big, the exponential's 2 u and the value scale's product u. Sums over
    blocks, units and lanes: one rounding of each of three products a block
    joined, 4 u (blocks + units + 8), for the numerator and the denominator
    each. The quotient: 3 u, then the type.

    Fixed point: a position's weight p times its value scale is cut at 2^-30 of a
    power of two that is at most twice the block's largest such product, itself
    at most P |v|max / 127 with P the block's largest probability: times a code, at
    most 2^-29 P |v|max. 64 positions: 2^-23 P |v|max; the P of all blocks sum to at
    most 1. So 2 u |v|max, whatever the output's own size (`mass` holds |v|max
    beside sum p |v|)."""
    u = 2.0 ** -24
    mass, top = mass
    blocks = length / 64 + 64 + 8
    return (u * (2 * (0.7 * 9 * big + 3) + 2 * 4 * blocks + 3)) * mass + 2 * u * top + HALF[dtype] * 1.01 * want.abs() + \
        (2.0 ** -24 if dtype == torch.float16 else 1e-30)


def run_attention(lens, counts, nh, nkv, hd, dtype=torch.float32, hidden=None, scale=None, seed=0, qscale=1.0, check=True,
                  **kw):
    pages = make_cache(lens, nkv, hd, seed=seed)
    k, v = fill(pages, lens, nkv, hd, seed=seed)
    q = rnd(sum(counts), nh, hd, seed=seed + 7, dtype=dtype, scale=qscale)
    hid = None if hidden is None else hidden.to(DEV)
    out = q8.attention(q.to(DEV), pages, i32(lens), starts(counts), max(counts), max(lens), scale=scale, hidden=hid, **kw)
    assert out.dtype == dtype and out.shape == q.shape
    kd, vd = values(k), values(v)
    sc = hd ** -0.5 if scale is None else scale
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        k0 = sum(lens[:i])
        if c and check:
            want, big, mass = ref_attention(q[at:at + c], kd[k0:k0 + n], vd[k0:k0 + n], list(range(n - c, n)),
                                            None if hidden is None else hidden[i], sc)
            got = out[at:at + c].cpu().double()
            far = (got - want).abs() - tolerance(dtype, n, big, mass, want)
            assert (far <= 0).all(), (i, n, c, float(far.max()), float((got - want).abs().max()))
        at += c
    return q, pages, out


@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (32, 8, 64), (8, 2, 128), (4, 2, 16), (3, 3, 40), (5, 1, 64), (14, 2, 80),
                                       (16, 2, 96), (2, 1, 1), (10, 1, 200), (4, 1, 256), (48, 1, 64)])
def test_attention_one_row_each(nh, nkv, hd):
    lens = [1, 2, 63, 64, 65, 127, 128, 129, 255, 300, 777]
    run_attention(lens, [1] * len(lens), nh, nkv, hd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (8, 2, 128), (4, 2, 16), (5, 1, 72), (8, 1, 64), (4, 4, 256), (14, 2, 192)])
def test_attention_rows_of_prompts(nh, nkv, hd, dtype):
    run_attention([70, 1, 200, 64, 150], [70, 1, 33, 0, 3], nh, nkv, hd, dtype=dtype, seed=3)


@pytest.mark.parametrize("qscale", [0.0, 1e-30, 0.01, 20.0])
def test_attention_flat_and_sharp(qscale):
    run_attention([500, 90], [5, 90], 4, 2, 64, qscale=qscale, seed=5)


def test_attention_long_sequences_cross_unit_lengths():
    # units of 128 positions up to 8,192, then 256, then 384: one row, and rows around the borders
    run_attention([20000, 8193, 8192], [1, 1, 1], 4, 1, 64)
    run_attention([8200], [20], 3, 1, 64, seed=2)
    run_attention([16390], [12], 8, 1, 64, seed=2)


def test_attention_hidden_positions():
    lens, counts = [130, 70, 300, 64, 5], [130, 1, 7, 64, 5]
    h = torch.rand(5, 310, generator=torch.Generator().manual_seed(1)) < 0.4
    h[1] = True         # sees nothing
    h[3, :40] = True    # its first rows see nothing
    for hidden in (h, h.to(torch.uint8) * 200, h[:, :70], h[:, :3], h.new_zeros(5, 0)):
        _, _, out = run_attention(lens, counts, 6, 2, 64, hidden=hidden.contiguous(), seed=4)
        if hidden.shape[1] >= 70:
            assert not out[130:131].any()
    wide = torch.zeros(5, 400, dtype=torch.bool, device=DEV)
    wide[:, :310] = h.to(DEV)
    q, pages, out = run_attention(lens, counts, 6, 2, 64, hidden=h, seed=4)
    again = q8.attention(q.to(DEV), pages, i32(lens), starts(counts), 130, 300, hidden=wide[:, :310])
    assert torch.equal(out, again)


def test_attention_does_not_see_what_it_must_not():
    """NaN in hidden places, in later positions, in the rest of a page and in pages of nobody changes nothing."""
    lens, nh, nkv, hd = [100, 140], 6, 2, 64
    pages = make_cache(lens, nkv, hd)  # its scales are NaN wherever nothing is written
    k, v = fill(pages, lens, nkv, hd)
    q = rnd(30, nh, hd, seed=9).to(DEV)
    h = torch.zeros(2, 140, dtype=torch.uint8, device=DEV)
    h[0, [3, 64, 99]] = 1
    h[1, 10:80] = 1
    args = (i32(lens), starts([10, 20]), 20, 140)
    want = q8.attention(q, pages, *args, hidden=h)
    assert torch.isfinite(want).all()
    bad = q8.Pages(*[t.clone() for t in pages])
    for i in range(2):
        for t in h[i].nonzero().flatten().tolist():
            p = int(pages.table[i, t // 64])
            bad.key_scale[p, :, t % 64] = math.nan
            bad.value_scale[p, :, t % 64] = math.inf
            bad.keys[p, :, t % 64] = 127
            bad.values[p, :, :, t % 64] = -128
    assert torch.equal(q8.attention(q, bad, *args, hidden=h), want)
    # a position that is seen: every later row of its heads is NaN, the earlier ones are not
    for scales in ("key_scale", "value_scale"):
        bad = q8.Pages(*[t.clone() for t in pages])
        getattr(bad, scales)[int(pages.table[0, 1]), 1, 95 - 64] = math.nan
        out = q8.attention(q, bad, *args, hidden=h)
        assert torch.isnan(out[5:10, 3:]).all() and torch.equal(out[:5], want[:5]) and torch.equal(out[5:10, :3], want[5:10, :3])
        assert torch.equal(out[10:], want[10:])
    # a query that is not finite is NaN, the others of its tile are not
    nan_q = q.clone()
    nan_q[4, 2, 7], nan_q[12, 0, 0] = math.nan, math.inf
    out = q8.attention(nan_q, pages, *args, hidden=h)
    bad_rows = torch.zeros(30, nh, dtype=torch.bool)
    bad_rows[4, 2] = bad_rows[12, 0] = True
    assert torch.isnan(out.cpu()[bad_rows]).all() and torch.equal(out.cpu()[~bad_rows], want.cpu()[~bad_rows])


def test_attention_sinks_keep_the_small_probabilities():
    """One score far above many small ones, whose values are all that counts: f32's accuracy, not the largest's."""
    n, hd = 3000, 64
    k, v = rnd(n, 1, hd, seed=1), rnd(n, 1, hd, seed=2)
    q = torch.zeros(1, 1, hd)
    q[0, 0, 0] = 8.0
    k[:, 0, 0] = 0
    k[5] = 0
    k[5, 0, 0] = 12.0  # score 96 * scale
    v[5] = 0
    pages = make_cache([n], 1, hd)
    q8.kv_write(pages, k.to(DEV), v.to(DEV), i32([n]), starts([n]), n)
    for scale in (0.0625, 0.1, 0.15):
        out = q8.attention(q.to(DEV), pages, i32([n]), starts([1]), 1, n, scale=scale).cpu().double()
        want, big, mass = ref_attention(q, values(k), values(v), [n - 1], None, scale)
        assert float((out - want).norm() / want.norm()) < 2e-5


def test_attention_most_len_bad_pages_and_rows_before_the_start():
    lens, nh, nkv, hd = [200, 90], 4, 2, 64
    pages = make_cache(lens, nkv, hd)
    k, v = fill(pages, lens, nkv, hd)
    kd, vd = values(k), values(v)
    q = rnd(4, nh, hd, seed=3)
    sc = hd ** -0.5

    def check(out, i, row, n, hidden=None):
        k0 = sum(lens[:i])
        want, big, mass = ref_attention(q[row:row + 1], kd[k0:k0 + n], vd[k0:k0 + n], [n - 1], hidden, sc)
        assert ((out[row:row + 1].cpu().double() - want).abs() <= tolerance(torch.float32, n, big, mass, want)).all()

    out = q8.attention(q[:2].to(DEV), pages, i32(lens), most_len=70)  # positions behind it are not attended to
    check(out, 0, 0, 70)
    check(out, 1, 1, 70)
    table = pages.table.clone()
    table[0, 1], table[1, 0] = 10 ** 6, -1
    holes = pages._replace(table=table)
    out = q8.attention(q[:2].to(DEV), holes, i32(lens))
    h = torch.zeros(2, 200)
    h[0, 64:128], h[1, :64] = 1, 1
    check(out, 0, 0, 200, h[0])
    check(out, 1, 1, 90, h[1])
    table[:] = -1
    assert not q8.attention(q[:2].to(DEV), holes._replace(table=table), i32(lens)).any()
    # a length of 0 and a row before position 0 see nothing; longer than the table: what there is
    out = q8.attention(q.to(DEV), pages, i32([0, 2]), starts([1, 3]), 3, 200)
    assert not out[:2].any()
    check(out, 1, 2, 1)
    check(out, 1, 3, 2)
    narrow = pages._replace(table=pages.table[:, :1].contiguous())
    check(q8.attention(q[:2].to(DEV), narrow, i32(lens)), 0, 0, 64)
    # rows of no sequence are left as they were
    into = torch.full((4, nh, hd), 3.0, device=DEV)
    got = q8.attention(q.to(DEV), pages, i32(lens), i32([1, 2, 3]), 1, 200, out=into)
    assert got is into and (into[0] == 3).all() and (into[3] == 3).all()
    check(into, 0, 1, 200)
    check(into, 1, 2, 90)
    assert not q8.attention(q.to(DEV), pages, i32(lens), i32([0, 2, 2]), 2, 200)[2:].any()
    assert q8.attention(q[:0].to(DEV), pages, i32(lens), i32([0, 0, 0])).shape == (0, nh, hd)


def test_attention_strides_and_types_of_a_fused_projection():
    """q, k and v as slices of one [rows, (nh + 2 nkv) hd] tensor, out a slice too."""
    nh, nkv, hd, lens, counts = 9, 3, 64, [40, 100], [40, 100]
    rows = sum(lens)
    for dtype in TYPES:
        y = rnd(rows, (nh + 2 * nkv) * hd, seed=3, dtype=dtype).to(DEV)
        q = y[:, :nh * hd].view(rows, nh, hd)
        k = y[:, nh * hd:(nh + nkv) * hd].view(rows, nkv, hd)
        v = y[:, (nh + nkv) * hd:].view(rows, nkv, hd)
        pages = make_cache(lens, nkv, hd)
        q8.kv_write(pages, k, v, i32(lens), starts(counts), 100)
        into = torch.zeros(rows, nh * hd + 64, dtype=dtype, device=DEV)
        q8.attention(q, pages, i32(lens), starts(counts), 100, 100, out=into[:, :nh * hd].view(rows, nh, hd))
        plain = make_cache(lens, nkv, hd)
        q8.kv_write(plain, k.contiguous(), v.contiguous(), i32(lens), starts(counts), 100)
        want = q8.attention(q.contiguous(), plain, i32(lens), starts(counts), 100, 100)
        assert torch.equal(into[:, :nh * hd].view(rows, nh, hd), want) and not into[:, nh * hd:].any()


@pytest.mark.parametrize("nh,nkv,hd,n", [(9, 3, 64, 200), (8, 2, 128, 140), (5, 1, 80, 300), (32, 8, 64, 333)])
def test_attention_rows_are_the_same_in_every_call(nh, nkv, hd, n):
    """A prompt at once, in pieces, row by row, beside other sequences, split over
    workgroups or not: the same bits."""
    pages = make_cache([n, 70], nkv, hd)
    fill(pages, [n, 70], nkv, hd)
    q = rnd(n + 70, nh, hd, seed=5).to(DEV)
    one = q8.Pages(*pages[:4], pages.table[:1].contiguous())
    all_rows = q8.attention(q[:n], one, i32([n]), starts([n]), n, n)
    both = q8.attention(q, pages, i32([n, 70]), starts([n, 70]), n, n)
    assert torch.equal(both[:n], all_rows)
    for a, b in ((0, 1), (3, 50), (50, 51), (60, n), (n - 1, n)):
        assert torch.equal(q8.attention(q[a:b], one, i32([b]), starts([b - a]), b - a, b), all_rows[a:b])
        assert torch.equal(q8.attention(q[a:b], one, i32([b]), starts([b - a])), all_rows[a:b])
    many = q8.Pages(*pages[:4], pages.table[:1].expand(400, -1).contiguous())  # too many rows to be split
    pos = torch.arange(400) % n
    out = q8.attention(q[pos.to(DEV)], many, i32((pos + 1).tolist()), most_len=n)
    assert torch.equal(out, all_rows[pos.to(DEV)])


def test_attention_long_rows_are_the_same_split_or_not():
    n, nh, nkv, hd = 8300, 4, 2, 64
    pages = make_cache([n], nkv, hd)
    fill(pages, [n], nkv, hd)
    pos = torch.cat([torch.arange(8150, 8300), torch.tensor([0, 63, 64, 4000])])
    q = rnd(len(pos), nh, hd, seed=2).to(DEV)
    rep = 6
    many = q8.Pages(*pages[:4], pages.table.expand(len(pos) * rep, -1).contiguous())
    out = q8.attention(q.repeat(rep, 1, 1), many, i32((pos + 1).repeat(rep).tolist()), most_len=n)
    assert torch.equal(out[:len(pos)], out[-len(pos):])
    for i in (0, 41, 42, 43, 149, 150, 153):
        one = q8.attention(q[i:i + 1], pages, i32([int(pos[i]) + 1]), most_len=n)
        assert torch.equal(one, out[i:i + 1]), i
    rows = q8.attention(q[:150], pages, i32([n]), starts([150]), 150, n)
    assert torch.equal(rows, out[:150])


@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 128), (16, 2, 64), (8, 2, 128)])
def test_attention_units_of_a_workgroup_are_the_same_in_one_piece(nh, nkv, hd):
    """Few sequences of 16 units, which share a workgroup, and many."""
    lens = [2048, 1921, 700]
    q, pages, out = run_attention(lens, [1, 1, 1], nh, nkv, hd, seed=2)
    rep = 400
    many = q8.Pages(*pages[:4], pages.table.repeat(rep, 1))
    got = q8.attention(q.repeat(rep, 1, 1).to(DEV), many, i32(lens * rep), most_len=2048)
    assert torch.equal(got, out.repeat(rep, 1, 1))


def test_attention_of_a_long_prompt_is_its_rows():
    n, nh, nkv, hd = 1100, 32, 8, 128
    pages = make_cache([n], nkv, hd)
    fill(pages, [n], nkv, hd)
    q = rnd(n, nh, hd, seed=4).to(DEV)
    out = q8.attention(q, pages, i32([n]), starts([n]), n, n)
    for a, b in ((0, 3), (500, 540), (1024, 1025), (n - 1, n)):
        assert torch.equal(q8.attention(q[a:b], pages, i32([b]), starts([b - a]), b - a, b), out[a:b])


def test_rows_of_a_call_without_sequences_are_zeros():
    pages = make_cache([100], 2, 40)
    q = rnd(5, 4, 40).to(DEV)
    none = pages._replace(table=torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    for p, n, start in ((none, i32([]), i32([0])), (pages, i32([100]), i32([2, 2]))):
        for dtype in TYPES:
            junk = torch.full((5, 4, 40), math.nan, dtype=dtype, device=DEV)  # what a fresh output may hold
            del junk
            assert not q8.attention(q.to(dtype), p, n, start, 0).any()
            assert not q8.attention(q.to(dtype), p, n, start, 5).any()
            for most in (0, 5):
                k, v = q8.kv_read(p, n, start, 5, 40, most, dtype)
                assert not k.any() and not v.any()
        keep = q.clone()
        q8.attention(q, p, n, start, 0, out=keep)
        assert torch.equal(keep, q)


def test_attention_refuses():
    pages = make_cache([100], 2, 64)
    q = rnd(1, 4, 64).to(DEV)
    n = i32([100])
    for bad in (lambda: q8.attention(q[:, :3], pages, n), lambda: q8.attention(q, pages, n, most_rows=2)):
        with pytest.raises((ValueError, G.DeferGpuError)):
            bad()
    for bad in (lambda: q8.attention(q[..., :63].transpose(1, 2), pages, n), lambda: q8.attention(q, pages, n.long()),
                lambda: q8.attention(q.double(), pages, n), lambda: q8.attention(q, pages, n.cpu()),
                lambda: q8.attention(rnd(1, 4, 65).to(DEV), pages, n), lambda: q8.attention(q, pages, i32([1, 2])),
                lambda: q8.attention(q, pages, n, hidden=torch.zeros(1, 100, device=DEV)),
                lambda: q8.attention(q, pages._replace(keys=pages.keys[:1]), n),
                lambda: q8.attention(q, pages._replace(values=pages.values.transpose(2, 3)), n),
                lambda: q8.attention(rnd(3, 4, 64).to(DEV), pages, n)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ streams, graphs, a layer

def layer(x, res, w, pages, lens, start, most, most_len, hidden=None):
    """One attention block on 8-bit weights and cache, every operator once."""
    nh, nkv, hd = w["heads"]
    z, c, s = q8.rms_norm(x, w["norm"], 1e-5, residual=res)
    y = q8.linear(c, s, *w["qkv"])
    rows = len(x)
    q = y[:, :nh * hd].view(rows, nh, hd)
    k = y[:, nh * hd:(nh + nkv) * hd].view(rows, nkv, hd)
    v = y[:, (nh + nkv) * hd:].view(rows, nkv, hd)
    q8.kv_write(pages, k, v, lens, start, most)
    o = q8.attention(q, pages, lens, start, most, most_len, hidden=hidden)
    return z, q8.linear(*q8.quantize(o.view(rows, nh * hd)), *w["o"])


def layer_weights(h, nh, nkv, hd, seed=0):
    w = {"heads": (nh, nkv, hd), "norm": (1 + rnd(h, seed=seed) / 10).to(DEV)}
    w["qkv"] = q8.quantize((rnd((nh + 2 * nkv) * hd, h, seed=seed + 1) / math.sqrt(h)).to(DEV))
    w["o"] = q8.quantize((rnd(h, nh * hd, seed=seed + 2) / math.sqrt(nh * hd)).to(DEV))
    return w


def test_a_layer_against_the_formulas():
    """The operators in a row, as a decoder layer uses them: a prompt, then a token,
    against 64-bit formulas that round to codes at the same places."""
    h, nh, nkv, hd, n = 576, 9, 3, 64, 77
    w = layer_weights(h, nh, nkv, hd)
    x, r = rnd(n, h, seed=4), rnd(n, h, seed=5)
    pages = make_cache([n], nkv, hd)
    z1, y1 = layer(x[:-1].to(DEV), r[:-1].to(DEV), w, pages, i32([n - 1]), starts([n - 1]), n - 1, n)
    z2, y2 = layer(x[-1:].to(DEV), r[-1:].to(DEV), w, pages, i32([n]), starts([1]), 1, n)
    got = torch.cat([y1, y2]).cpu().double()
    z = (x + r)
    assert torch.equal(torch.cat([z1, z2]).cpu(), z)
    d = z.double()
    norm = values((d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5)) * w["norm"].cpu().double())
    deq = lambda p: p[0].cpu().double() * p[1].cpu().double()[:, None]  # noqa: E731
    y = (norm @ deq(w["qkv"]).t())
    q, k, v = y[:, :nh * hd].view(n, nh, hd), y[:, nh * hd:(nh + nkv) * hd].view(n, nkv, hd), y[:, (nh + nkv) * hd:].view(n, nkv, hd)
    o, _, _ = ref_attention(q, values(k), values(v), list(range(n)), None, hd ** -0.5)
    want = values(o.reshape(n, nh * hd)) @ deq(w["o"]).t()
    # f32 roundings before a quantiser move a code where a quotient is next to a half: one step of
    # a row's scale (max / 127) in a few of its nh * hd = 576 places. 1 % of the places (a rounding of
    # 1e-6 of a step's 1/2 reaches far fewer) gives sqrt(5.76) steps of max / 127 ~ 4 / 127 of a value.
    assert float((got - want).norm() / want.norm()) < math.sqrt(5.76) * 4 / 127 / math.sqrt(576)


def test_a_layer_in_a_graph_and_on_streams():
    h, nh, nkv, hd, n = 256, 8, 2, 64, 300
    w = layer_weights(h, nh, nkv, hd)
    lens, most_len = i32([n, 9, 130]), n
    prompts = [n - 1, 8, 129]
    x = rnd(3, h, seed=8).to(DEV)
    r = rnd(3, h, seed=9).to(DEV)

    def fresh(seed):
        pages = make_cache([n, 9, 130], nkv, hd, seed=1)
        fill(pages, [n, 9, 130], nkv, hd, seed=seed)
        return pages

    def eager(pages, x):
        return layer(x, r, w, pages, lens, None, 1, most_len)

    assert prompts
    pages = fresh(1)
    want = {s: eager(fresh(1), x * s) for s in (1.0, 0.5, -2.0)}
    # captured once, replayed with other inputs and eager work between
    gx = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager(pages, gx)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gz, gy = eager(pages, gx)
    for s in (1.0, 0.5, -2.0, 1.0):
        gx.copy_(x * s)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(gz, want[s][0]) and torch.equal(gy, want[s][1]), s
        assert torch.equal(eager(fresh(1), x)[1], want[1.0][1])
    # two streams at once, each with a cache of its own
    caches, outs = [fresh(1), fresh(1)], [None, None]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = eager(caches[i], x * (1.0 if i == 0 else 0.5))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][1], want[1.0][1]) and torch.equal(outs[1][1], want[0.5][1])


def test_calls_return_the_callers_tensors_and_keep_nothing():
    nh, nkv, hd = 4, 2, 64
    lens = [3000, 40]
    pages = make_cache(lens, nkv, hd)
    k, v = (t.to(DEV) for t in fill(pages, lens, nkv, hd))
    x, w, q = rnd(2, 64).to(DEV), rnd(64).to(DEV), rnd(2, nh, hd).to(DEV)
    n, start = i32(lens), starts([1, 1])
    refs = (x, w, q, n, start, k, v, *pages)

    def calls():
        z, c, s = q8.rms_norm(x, w, 1e-5)
        assert z is x
        into = torch.empty_like(x)
        assert q8.rms_norm(x, w, 1e-5, residual=x, out=into)[0] is into
        out = torch.empty_like(q)
        assert q8.attention(q, pages, n, start, 1, out=out) is out
        q8.attention(q, pages, n, start, 1, 3000)
        q8.linear(c, s, c, s, torch.float16)
        q8.kv_write(pages, k, v, n, starts(lens), 3000)
        q8.kv_read(pages, n, start, 2, hd, 1)
        for bad in (lambda: q8.attention(q, pages, n, start, 7), lambda: q8.attention(q, pages, n, start, 1, 1 << 31),
                    lambda: q8.attention(q, pages, n, start, 1, hidden=x), lambda: q8.kv_read(pages, n, start, 2, 65),
                    lambda: q8.kv_read(pages, n, start, -1, hd), lambda: q8.kv_read(pages[:4], n, start, 2, hd),
                    lambda: q8.linear(c, s, c, s, torch.int8), lambda: q8.linear(c, s, c, s, "float32")):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(TypeError):
            q8.attention(q, pages, n, start, 1.5)
        with pytest.raises(G.DeferGpuError):
            q8.rms_norm(x, w, float("nan"))

    calls()
    torch.cuda.synchronize()
    held, counts = torch.cuda.memory_allocated(), [sys.getrefcount(t) for t in refs]
    for _ in range(20):
        calls()
    assert torch.cuda.memory_allocated() == held and [sys.getrefcount(t) for t in refs] == counts


def test_calls_from_two_threads_on_two_streams():
    import threading

    x, w = rnd(64, 512, seed=1).to(DEV), rnd(300, 512, seed=2).to(DEV)
    wc, ws = q8.quantize(w)
    want = q8.linear(*q8.quantize(x), wc, ws)
    torch.cuda.synchronize()
    bad = []

    def work(stream):
        with torch.cuda.stream(stream):
            for _ in range(200):
                y = q8.linear(*q8.quantize(x), wc, ws)
            stream.synchronize()
            if not torch.equal(y, want):
                bad.append(stream)

    ts = [threading.Thread(target=work, args=(torch.cuda.Stream(),)) for _ in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad



def test_large_offsets():
    """Pages and rows whose byte offsets pass 32 bits."""
    heads, hd = 8, 128
    per = heads * 64 * 128
    pool = (1 << 32) // per + 40  # keys of over 4 GiB
    table = torch.tensor([[pool - 1, 3, pool - 2]], dtype=torch.int32, device=DEV)
    pages = q8.Pages(torch.empty(pool, heads, 64, 128, dtype=torch.int8, device=DEV),
                     torch.empty(pool, heads, 128, 64, dtype=torch.int8, device=DEV),
                     torch.empty(pool, heads, 64, device=DEV), torch.empty(pool, heads, 64, device=DEV), table)
    n = 150
    k, v = rnd(n, heads, hd, seed=1), rnd(n, heads, hd, seed=2)
    q8.kv_write(pages, k.to(DEV), v.to(DEV), i32([n]), starts([n]), n)
    rk, rv = q8.kv_read(pages, i32([n]), starts([n]), n, hd)
    assert ((rk.cpu().double() - values(k)).abs() <= 1e-7 * values(k).abs()).all()
    assert ((rv.cpu().double() - values(v)).abs() <= 1e-7 * values(v).abs()).all()
    q = rnd(2, 16, hd, seed=3)
    out = q8.attention(q.to(DEV), pages, i32([n]), starts([2]), 2, n)
    want, big, mass = ref_attention(q, values(k), values(v), [n - 2, n - 1], None, hd ** -0.5)
    assert ((out.cpu().double() - want).abs() <= tolerance(torch.float32, n, big, mass, want)).all()
    del pages, rk, rv
    # a weight of over 4 GiB
    m, kk = 40000, 110000
    w = torch.empty(m, kk, dtype=torch.int8, device=DEV)
    w[-200:] = i8(200, kk, seed=4).to(DEV)
    x = i8(2, kk, seed=5)
    y = q8.linear(x.to(DEV), torch.ones(2, device=DEV), w, torch.ones(m, device=DEV))
    check_linear(x, torch.ones(2), w[-200:].cpu(), torch.ones(200), torch.float32, y[:, -200:])
