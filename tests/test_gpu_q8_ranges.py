"""GPU: the 8-bit operators at the ends of their value types' ranges, against
plain 64-bit implementations on the CPU."""
import numpy as np
import pytest
import torch

from defer_amd import q8

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
