"""The operators for drafted tokens at operands where a definition and a shortcut part: zeros kept from pages of large scales; norms beside the
middle of two fp32 numbers."""
import math
from fractions import Fraction

import numpy as np
import pytest

import drafts_ref as D
import fp8_ref as F
import test_gpu_drafts as T
import test_gpu_fp8_serving as S
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu


# ---- zeros from pages of large scales --------------------------------------------------------------
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("octave", [20, 28, 40, 110])
def test_kept_zeros_stay_zeros(ctx, d, octave):
    """A token of zeros on a page of scale 2^octave moves to a page of zeros, whose scale is 2^-100: their ratio is beyond fp32 from 2^28 on.
    A second one moves beside a token that is not 0."""
    past, new = 60, 9                                                         # rows 4 .. are on the second page
    k = np.zeros((past + new, 2, d), np.float32)
    k[-1, 0] = np.float32(448 * 2.0 ** octave)                                # (of the first head; the second page of the other is zeros too)
    table, lens, starts = np.array([[1, 0]], np.int32), np.array([past + new], np.int32), np.array([0, past + new], np.int32)
    for other in (0.0, 3.0):
        k[past + 5] = other
        k[past + 5, :, 1] = 0
        c = F.Cache(2, 2, d)
        c.append(k, -k, table, lens, starts)
        device = S.on_device(ctx, c)
        rows, path, count = np.array([0, new], np.int32), np.array([0, 4, 5, 6] + [-1] * 5, np.int32), np.array([3], np.int32)
        H.cache_keep(ctx, device, *T.up(ctx, table, lens, rows, path, count))
        D.keep(c, table, lens, rows, path, count)
        S.check_cache(device, c)
        assert not np.any((device.k.get_data()[1] & 0x7f) == 0x7f)


# ---- norms beside the middle of two fp32 numbers ------------------------------------------------------
def squares_of(n):
    """Four whole numbers whose squares add up to n."""
    a = math.isqrt(n)
    while True:
        b = math.isqrt(n - a * a)
        while b >= 0:
            left = n - a * a - b * b
            c = math.isqrt(left)
            while c * c * 2 >= left and c >= 0:
                e = math.isqrt(left - c * c)
                if e * e == left - c * c:
                    return a, b, c, e
                c -= 1
            b -= 1
            if math.isqrt(n - a * a) - b > 8:
                break
        a -= 1


def rows_beside_a_middle(d, seed):
    """(rows of keys, gamma): the mean of a row's squares in 64 bits, and with it the fp32 factor 1 / sqrt(mean), depends on the order of addition.

    Element 0 is near 1; elements 1, 2, 3 and 12 bring the sum S of a row to r units of 2^-52 from where the factor crosses the middle between two fp32
    numbers, r = -70 .. 69 from row to row.  Squares of 0.9999 / 2 such units lie in pieces of four that the two orders bring to S in different company:
    alone they are rounded away, two of them together count as one unit.  gamma takes the two possible results of element 0 to both sides of 272, the
    middle between two e4m3 values."""
    rng = np.random.default_rng(seed)
    unit = Fraction(1, 2 ** 52)
    while True:
        low = np.float32(rng.uniform(8.2, 11.2)) if d == 128 else np.float32(rng.uniform(5.8, 7.9)) if d == 64 else np.float32(rng.uniform(4.1, 5.6))
        high = np.nextafter(low, np.float32(np.inf))
        middle = (Fraction(float(low)) + Fraction(float(high))) / 2
        target = int(Fraction(d) / (middle * middle) / unit)                  # S in units; 1 <= S < 2
        x0 = np.nextafter(np.float32(math.sqrt(target * 2.0 ** -52)), np.float32(0))
        x0 = np.nextafter(x0, np.float32(0))
        left = target - Fraction(float(x0)) ** 2 / unit
        if left.denominator != 1 or left < 200:
            continue
        for _ in range(4000):
            gamma0 = np.float32(272 / (float(x0) * float(middle)) * (1 + rng.uniform(-2, 2) * 2.0 ** -23))
            if (x0 * low) * gamma0 <= 272 < (x0 * high) * gamma0:
                break
        else:
            continue
        rows = np.zeros((140, d), np.float32)
        rows[:, 0] = x0
        for i in range(len(rows)):
            rows[i, [1, 2, 3, 12]] = np.array(squares_of(int(left) + i - 70), np.float64) * 2.0 ** -26
        half = np.float32(math.sqrt(0.9999 * 2.0 ** -53))
        for piece in {32: [1, 2, 5, 6], 64: [1, 9, 2, 10, 4, 12], 128: [1, 17, 2, 18, 4, 20, 8, 24]}[d]:
            rows[:, 4 * piece + 1] = half
        gamma = np.ones(d, np.float32)
        gamma[0] = gamma0
        return rows, gamma


@pytest.mark.parametrize("d,rotary,interleaved", [(32, 32, False), (32, 32, True), (32, 20, False), (32, 0, False), (64, 64, False), (64, 64, True), (64, 22, False), (64, 0, False),
                                                  (128, 128, False), (128, 64, False), (128, 128, True), (128, 30, False), (128, 0, False)])
def test_append_rope_adds_squares_as_rope_does(ctx, d, rotary, interleaved):
    """The cache holds the bits of wdh_rope and wdh_cache_append where the order of a sum of 64 bits decides about them (rotation by no angle)."""
    rows, gamma = rows_beside_a_middle(d, d)
    n = len(rows)
    table, lens, starts = np.arange(3, dtype=np.int32)[None], np.array([n], np.int32), np.array([0, n], np.int32)
    cos, sin = (np.ones((n, rotary // 2), np.float32), np.zeros((n, rotary // 2), np.float32)) if rotary else (None, None)
    dk, dt, dl, ds, dc, dn, dg = T.up(ctx, rows, table, lens, starts, cos, sin, gamma)
    one, two = (S.on_device(ctx, F.Cache(3, 1, d)) for _ in range(2))
    H.cache_append_rotary(ctx, one, dk, dk, dt, dl, ds, dc, dn, None, dg, interleaved, 0.0)
    turned = H.rotary_embedding(ctx, dk, dc, dn, None, 1, d, q_scale=dg, interleaved=interleaved, epsilon=0.0)
    H.cache_append(ctx, two, turned, dk, dt, dl, ds)
    first = turned.get_data()[:, 0]
    assert np.any(first <= 272) and np.any(first > 272)                       # (the rows are on both sides of the middle)
    assert np.array_equal(one.k_scales.get_data(), two.k_scales.get_data())
    assert np.array_equal(one.k.get_data(), two.k.get_data())
