"""GPU: the sines and cosines that kv_append turns rows by have 64 bits' accuracy, seen where a
rotation takes nearly all of a value away."""
import random
from fractions import Fraction

import pytest
import torch

from defer_amd import q8
from test_gpu_draft import PI
from test_gpu_q8 import DEV, i32, make_cache, starts

pytestmark = pytest.mark.gpu
BITS = 120


def sin_cos(turns):
    """Of a fraction of turns, as whole multiples of 2^-120: the series, in whole numbers."""
    quarter = round(4 * turns)
    x = int((turns - Fraction(quarter, 4)) * 2 * PI * 2 ** BITS)
    s, c, term, n = 0, 0, 1 << BITS, 0
    while term:
        if n % 2:
            s += term if n % 4 == 1 else -term
        else:
            c += term if n % 4 == 0 else -term
        n += 1
        term = ((term * x) >> BITS) // n
    return [(s, c), (c, -s), (-s, -c), (-c, s)][quarter % 4]


def test_series():
    for t in (Fraction(1, 8), Fraction(-1, 8), Fraction(1, 12), Fraction(3, 7), Fraction(5, 6), Fraction(123456, 1001)):
        s, c = sin_cos(t)
        assert abs(s * s + c * c - (1 << 2 * BITS)) < 1 << BITS + 8
    assert abs(sin_cos(Fraction(1, 12))[0] - (1 << BITS - 1)) < 256 and abs(sin_cos(Fraction(2, 3))[1] + (1 << BITS - 1)) < 256


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,odd", [(64, False), (64, True), (200, False)])
def test_append_turns_values_to_nearly_nothing(hd, odd, interleaved):
    """(a, b) = r (sin, cos) in f32 becomes (about 2^-25 r, r). The angle is off by less than 2^-50 (turns up to 1 are
    rounded by 2^-54 or 2^-53, times 2 pi; the product with 2 pi and that constant by 2^-54 each), sine and cosine by a few
    roundings of 2^-54 besides: less than 2^-49 r of the result in all, which is then rounded to f32."""
    g = random.Random(hd)
    rows, half = 12, hd // 2
    freq = [g.uniform(0.1, 3) for _ in range(half)]
    pos = [0, 1, 2, 2 ** 31 - 1, -2 ** 31] + [g.randrange(1 << 20) for _ in range(rows - 5)]
    q = torch.zeros(rows, 1, hd, dtype=torch.float64)
    at = (lambda i: (2 * i, 2 * i + 1)) if interleaved else (lambda i: (i, i + half))
    angles = {}
    for j in range(rows):
        for i in range(half):
            s, c = angles[j, i] = sin_cos(Fraction(freq[i]) * pos[j] / (2 * PI) % 1)
            r = g.uniform(0.5, 2)
            q[j, 0, at(i)[0]], q[j, 0, at(i)[1]] = r * s / 2 ** BITS, r * c / 2 ** BITS
    q = q.float()
    wide = torch.zeros(rows, 1, hd + 1, device=DEV)
    wide[..., odd:hd + odd] = q.to(DEV)
    rot = q8.Rotary(torch.tensor(freq, dtype=torch.float64, device=DEV), interleaved)
    pages = make_cache([rows], 1, hd)
    x = wide[..., 1:] if odd else q.to(DEV)
    out = q8.kv_append(pages, x, x, x, i32([rows]), rot, starts([rows]), rows, position=i32(pos)).cpu()
    worst = 0.0
    for j in range(rows):
        for i in range(half):
            s, c = angles[j, i]
            a, b = (Fraction(float(q[j, 0, k])) for k in at(i))
            first, second = float((a * c - b * s) / 2 ** BITS), float((b * c + a * s) / 2 ** BITS)
            r = float(a * a + b * b) ** 0.5
            got = [float(out[j, 0, k]) for k in at(i)]
            for value, want in zip(got, (first, second)):
                off = (abs(value - want) - 2.0 ** -24 * abs(want)) / r
                worst = max(worst, off)
    assert worst <= 2.0 ** -49, worst
