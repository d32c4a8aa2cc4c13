"""GPU: the 8-bit operators at the ends of their value types' ranges, against
plain 64-bit implementations on the CPU."""
import numpy as np
import pytest
import torch

from defer_amd import q8
from test_gpu_q8 import i32, make_cache, ref_attention, rnd, starts, tolerance, values

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i8(*shape, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(-127, 128, shape, dtype=np.int8))


# ------------------------------------------------------------------ the product

# rows, channels, k: few rows, 64 x 64 tiles, unaligned rows
SIZES = [(1, 40, 4096), (33, 100, 4096), (130, 200, 4096), (70, 90, 4001)]


@pytest.mark.parametrize("rows,m,k", SIZES)
def test_linear_sums_times_a_large_row_scale(rows, m, k):
    """Sums of some 1e5 times a row scale of 1e34 and more pass f32's range; the
    values do not."""
    x, w = i8(rows, k, seed=1), i8(m, k, seed=2)
    acc = x.double() @ w.double().t()
    for a, b in ((1e34, 1e-20), (2e36, 1e-30), (1e34, 2.0 ** -107), (1e-20, 1e34), (2.0 ** 64, 3.0), (1.0001 * 2.0 ** 64, 3.0)):
        xs, ws = torch.full((rows,), a), torch.full((m,), b)
        y = q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV)).cpu().double()
        want = acc * xs.double()[:, None] * ws.double()
        # the sum to f32 and two products: half a step each
        assert ((y - want).abs() <= 3.03 * 2.0 ** -24 * want.abs()).all(), (a, b)
    xs, ws = torch.full((rows,), 1e34), torch.zeros(m)
    assert not q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV)).any()
    # a value that passes the range is infinite, one of a row that is not finite NaN
    xs[0] = float("nan")
    y = q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), torch.full((m,), 1e20, device=DEV)).cpu()
    assert torch.isnan(y[0]).all() and torch.isinf(y[1:][acc[1:] != 0]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_of_rows_quantised_from_large_values(dtype):
    """The same through the quantiser: rows of up to 1e37, weights of 1e-10."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(20, 2000, generator=g).to(dtype) * 1e36, torch.randn(50, 2000, generator=g) * 1e-10
    (xc, xs), (wc, ws) = q8.quantize(x.to(DEV)), q8.quantize(w.to(DEV))
    y = q8.linear(xc, xs, wc, ws, dtype=dtype).cpu().double()
    want = (xc.cpu().double() @ wc.cpu().double().t()) * xs.cpu().double()[:, None] * ws.cpu().double()
    assert ((y - want).abs() <= (3.03 * 2.0 ** -24 + 1.01 * torch.finfo(dtype).eps / 2) * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,m,k", SIZES)
def test_linear_large_row_scales_in_every_type(rows, m, k, dtype):
    """Some rows of a tile over 2^64, some not: each as if it were alone."""
    x, w = i8(rows, k, seed=3), i8(m, k, seed=4)
    xs, ws = torch.full((rows,), 2.0 ** 70), torch.full((m,), 1.7 * 2.0 ** -82)
    xs[::3] = 1.3
    y = q8.linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), dtype=dtype)
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    tol = (3.03 * 2.0 ** -24 + 1.01 * torch.finfo(dtype).eps / 2) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((y.cpu().double() - want).abs() <= tol).all()
    for i in range(0, rows, 7):
        assert torch.equal(q8.linear(x[i:i + 1].to(DEV), xs[i:i + 1].to(DEV), w.to(DEV), ws.to(DEV), dtype=dtype), y[i:i + 1])


# ------------------------------------------------------------------ attention

def attend(lens, counts, nh, nkv, hd, dtype, kscale, qscale, hidden=None, loud=None):
    """Rows of each sequence's end against the formula; the queries, the pages and what came out."""
    pages = make_cache(lens, nkv, hd, seed=hd)
    k = (rnd(sum(lens), nkv, hd, seed=1) * kscale).to(dtype)
    if loud is not None:  # a few keys of their own size
        at, size = loud
        k[at] = (rnd(len(at), nkv, hd, seed=4) * size).to(dtype)
    v = rnd(sum(lens), nkv, hd, seed=2, dtype=dtype)
    q = (rnd(sum(counts), nh, hd, seed=3) * qscale).to(dtype)
    q8.kv_write(pages, k.to(DEV), v.to(DEV), i32(lens), starts(lens), max(lens))
    out = q8.attention(q.to(DEV), pages, i32(lens), starts(counts), max(counts), max(lens),
                       hidden=None if hidden is None else hidden.to(DEV))
    kd, vd, at = values(k), values(v), 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        k0 = sum(lens[:i])
        want, big, mass = ref_attention(q[at:at + c], kd[k0:k0 + n], vd[k0:k0 + n], list(range(n - c, n)),
                                        None if hidden is None else hidden[i], hd ** -0.5)
        got = out[at:at + c].cpu().double()
        assert torch.isfinite(got).all()
        far = (got - want).abs() - tolerance(dtype, n, big, mass, want)
        assert (far <= 0).all(), (i, float(far.max()))
        at += c
    return q, pages, out


# one row in one piece, in a workgroup's units, split over workgroups; a prompt
SPREAD = [([60, 100], [1, 1]), ([777], [1]), ([3000], [1]), ([200, 70], [200, 33])]
# keys' size, queries' size: products of some 1 to 10, the ends of f32's and bf16's range
FAR = [(1e32, 1e-32), (5e37, 2e-38), (1e26, 1e-25), (1e-26, 1e26), (2e-30, 1e30), (1.0, 1e-40), (1e-20, 1e-20)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (16, 2, 128), (3, 1, 40)])
@pytest.mark.parametrize("lens,counts", SPREAD)
def test_attention_of_large_and_small_keys(lens, counts, nh, nkv, hd, dtype):
    for kscale, qscale in FAR:
        attend(lens, counts, nh, nkv, hd, dtype, kscale, qscale)


@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (16, 2, 128), (2, 1, 256)])
def test_attention_of_a_few_large_keys_among_small_ones(nh, nkv, hd):
    """Rows before and behind them, hidden or not; each the same bits in any call."""
    n, at = 300, torch.tensor([3, 70, 131, 255])
    shown = torch.zeros(1, n, dtype=torch.bool)
    shown[0, 131] = True
    for hidden in (None, shown):
        for size, qscale in ((1e33, 1e-33), (1e37, 1e-36)):
            q, pages, out = attend([n], [n], nh, nkv, hd, torch.float32, 1e25, qscale, hidden, (at, size))
            h = None if hidden is None else hidden.to(DEV)
            for a, b in ((0, 3), (3, 4), (60, 80), (130, 133), (299, 300)):
                got = q8.attention(q[a:b].to(DEV), pages, i32([b]), starts([b - a]), b - a, b, hidden=h)
                assert torch.equal(got, out[a:b]), (a, b)


def test_attention_of_queries_of_every_size_in_a_tile():
    """One row large, one small, one not finite, one of zeros: each as if it were alone."""
    n, nh, nkv, hd = 130, 8, 2, 64
    pages = make_cache([n], nkv, hd)
    k, v = rnd(n, nkv, hd, seed=1), rnd(n, nkv, hd, seed=2)
    q8.kv_write(pages, k.to(DEV), v.to(DEV), i32([n]), starts([n]), n)
    q = rnd(12, nh, hd, seed=3)
    for i, size in enumerate((1e30, 1e-30, 1e37, 1e-38, 1e20, 1e-20, 2.0 ** 64, 2.0 ** -64, 1.0, 0.0)):
        q[i] *= size
    q[10, 0, 0], q[11, 3, 5] = float("inf"), float("nan")
    out = q8.attention(q.to(DEV), pages, i32([n]), starts([12]), 12, n)
    for i in range(12):
        one = q8.attention(q[i:i + 1].to(DEV), pages, i32([n - 11 + i]))
        assert torch.equal(torch.isnan(one), torch.isnan(out[i:i + 1]))
        assert torch.equal(one.nan_to_num(), out[i:i + 1].nan_to_num()), i
    assert torch.isnan(out[10, 0]).all() and torch.isnan(out[11, 3]).all() and torch.isfinite(out[:10]).all()
    assert torch.isfinite(out[10, 1:]).all() and torch.isfinite(out[11, :3]).all()
    kd, vd = values(k), values(v)
    for i in (1, 3, 5, 7, 8, 9):
        want, big, mass = ref_attention(q[i:i + 1], kd[:n - 11 + i], vd[:n - 11 + i], [n - 12 + i], None, hd ** -0.5)
        assert ((out[i:i + 1].cpu().double() - want).abs() <= tolerance(torch.float32, n, big, mass, want)).all(), i


@pytest.mark.parametrize("lens,counts", SPREAD)
def test_attention_of_scores_too_large_for_a_softmax(lens, counts):
    """Scores of 1e9 and more: the row's largest one takes all, on any size of either."""
    nh, nkv, hd = 6, 2, 64
    for kscale, qscale in ((1.0, 1e10), (1.0, 1e25), (1e15, 1e5), (1e15, 1e20), (1e-15, 1e30)):
        pages = make_cache(lens, nkv, hd, seed=1)
        k, v = rnd(sum(lens), nkv, hd, seed=1) * kscale, rnd(sum(lens), nkv, hd, seed=2)
        q = rnd(sum(counts), nh, hd, seed=3) * qscale
        q8.kv_write(pages, k.to(DEV), v.to(DEV), i32(lens), starts(lens), max(lens))
        out = q8.attention(q.to(DEV), pages, i32(lens), starts(counts), max(counts), max(lens)).cpu().double()
        kd, vd, at, sure = values(k), values(v), 0, 0
        for i, (n, c) in enumerate(zip(lens, counts)):
            k0 = sum(lens[:i])
            for j in range(c):
                m = n - c + j + 1
                for h in range(nh):
                    s = kd[k0:k0 + m, h // 3] @ q[at + j, h].double() * hd ** -0.5
                    s, order = s.sort(descending=True)
                    # a score is off by some 10 half steps of the largest, and by 2^-30 of each product's factors
                    if m == 1 or s[0] - s[1] > 100 + 2.0 ** -18 * s.abs().max():
                        want = vd[k0 + order[0], h // 3]
                        assert ((out[at + j, h] - want).abs() <= 2.0 ** -20 * want.abs().max()).all(), (kscale, qscale, i, j, h)
                        sure += 1
            at += c
        assert sure >= 0.9 * sum(counts) * nh


@pytest.mark.parametrize("nh,nkv,hd,lens,counts", [(4, 1, 64, [8200], [20]), (8, 2, 128, [8200], [9]), (8, 2, 192, [300, 70], [300, 70]),
                                                   (6, 3, 192, [700], [2]), (4, 1, 256, [300], [300]), (16, 2, 128, [1100], [1100])])
def test_attention_at_both_ends_across_units_and_head_sizes(nh, nkv, hd, lens, counts):
    for kscale, qscale in ((1e32, 1e-32), (1e-26, 1e26)):
        attend(lens, counts, nh, nkv, hd, torch.float32, kscale, qscale)
