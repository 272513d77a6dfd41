"""The operators for drafted tokens at operands where a definition and a shortcut part: zeros kept from pages of large scales; norms beside the
middle of two fp32 numbers; attention of trees over pages whose values differ in size, at scores of any size, and in 2-norm in every form."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import drafts_ref as D
import fp8_ref as F
import test_gpu_drafts as T
import test_gpu_fp8_edges as X
import test_gpu_fp8_serving as S
import tree_plan
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


# ---- attention over pages whose values differ in size ----------------------------------------------
def chain(n):
    return H.tree_mask(np.arange(-1, n - 1), np.array([0, n]))


@pytest.mark.parametrize("octaves", [0, 16, 30, 60, 82])
@pytest.mark.parametrize("new,heads,kv,d,large", [(1, 4, 2, 64, [0]), (7, 4, 1, 128, [3, 4]), (90, 4, 2, 64, [2]), (30, 4, 2, 32, [9]), (650, 64, 2, 64, [0]),
                                                  (650, 64, 2, 64, [3, 7]), (650, 64, 2, 64, [11]), (700, 32, 4, 128, [1]), (1300, 64, 2, 32, [0, 9])])
def test_values_of_pages_that_differ_in_size(ctx, new, heads, kv, d, large, octaves):
    """As of wdh_cache_attention, with its bound: rows of chains."""
    rng = np.random.default_rng(octaves)
    past = 640
    c, table, lens, starts, q = X.sized_pages(rng, new, past, heads, kv, d, large, octaves)
    want = X.attention(c, q, table[0], int(lens[0]), d ** -0.5)
    got = T.attend_tree(ctx, c, q, table, lens, starts, chain(new), np.float32(d ** -0.5))
    assert X.relative(got, want) <= 2.0 ** -20, (X.relative(got, want) * 2 ** 20)


@pytest.mark.parametrize("small,large,nats", [(-90, 110, 320), (-90, 110, 40), (-90, 110, 7), (-30, 100, 160), (0, 70, 60), (-95, -30, 30), (-20, 40, 0), (0, 50, 22)])
@pytest.mark.parametrize("new,heads,kv,d,pages", [(2, 4, 2, 64, [0]), (2, 4, 2, 64, [9]), (9, 4, 1, 128, [4, 5]), (50, 4, 2, 64, [0, 3]), (90, 4, 2, 32, [2]), (650, 64, 2, 64, [0, 5]),
                                                  (650, 64, 2, 64, [8])])
def test_pages_of_all_sizes_count_by_their_shares(ctx, new, heads, kv, d, pages, small, large, nats):
    """Some pages hold values of 2^large, the others of 2^small; the former's keys are `nats` below the latter's.  Which of them a row rests on goes by weight
    times value, and its sum of weights by the weights alone.

    The bound for scores of size one: see test_gpu_fp8_edges.test_values_of_pages_that_differ_in_size.  Here one product of a score is `nats`, alike for all keys of
    a page, so that what it is off shows in all of a row: 2^-23 by its query's parts, 2^-24 each by alpha, alpha log2(e) and the query times that (3 / 2^23 together), and
    2^-23 by each of the 2 d / 16 instructions that add to it (their additions need not round to nearest); in all nats (3 + d / 8) 2^-23 of a weight."""
    rng = np.random.default_rng(large - small)
    past = 640
    table, lens, starts, count = S.layout(rng, [new], [past])
    n = int(lens[0])
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((new, heads, d)).astype(np.float32)
    k[:, :, 0], q[:, :, 0] = 0, 16
    octave = np.full(n, small)
    for page in pages:
        at = slice(64 * page, 64 * page + 64)
        k[at, :, 0], octave[at] = -nats / 16 / d ** -0.5, large
    v *= np.float32(2) ** octave.astype(np.float32)[:, None, None]
    c = F.Cache(count, kv, d)
    c.append(k, v, table, lens, np.array([0, n]))
    want = X.attention(c, q, table[0], n, d ** -0.5)
    got = T.attend_tree(ctx, c, q, table, lens, starts, chain(new), np.float32(d ** -0.5))
    assert X.relative(got, want) <= 2.0 ** -20 + nats * (3 + d / 8) * 2.0 ** -23, (X.relative(got, want) * 2 ** 20)


@pytest.mark.parametrize("new,past,heads,kv,d", [(1, 900, 8, 2, 64), (60, 100, 4, 2, 128), (3, 3000, 2, 1, 128), (650, 100, 64, 2, 64), (700, 0, 32, 4, 128), (40, 200, 2, 2, 32)])
@pytest.mark.parametrize("size", [1e2, 3e3, 1e4, 1e5, 1e7, 1e9, 1e14])
def test_scores_of_any_size(ctx, new, past, heads, kv, d, size):
    """Where neighbouring fp32 numbers are further apart than the powers of two that weights are, rows rest on their largest score: the others
    are left far behind (rows whose two largest scores are not further apart than their errors are left out), on pages whose values are 2^5 times as
    large too (2^10 times what is 30 nats below: 2^-33)."""
    rng = np.random.default_rng(new)
    table, lens, starts, pages = S.layout(rng, [new], [past])
    n = int(lens[0])
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in range(2))
    c = F.Cache(pages, kv, d)
    c.append(k * np.float32(size), v, table, lens, np.array([0, n]))
    c.ks *= rng.uniform(0.5, 1, c.ks.shape).astype(np.float32)
    c.vs *= rng.uniform(0.5, 1, c.vs.shape).astype(np.float32) * np.float32(2) ** rng.integers(-5, 6, c.vs.shape).astype(np.float32)
    q = (rng.standard_normal((new, heads, d)) * size).astype(np.float32)
    keys, values = c.tokens(table[0], n)
    got = T.attend_tree(ctx, c, q, table, lens, starts, chain(new), 0.125)
    tried = 0
    for h in range(heads):
        kv_head = h // (heads // kv)
        t = q[:, h].astype(np.float64) @ keys[kv_head].T * 0.125
        t[np.arange(n) > np.arange(new)[:, None] + past] = -np.inf
        order = np.sort(t, 1)
        far = np.ones(new, bool) if n == 1 else order[:, -1] - order[:, -2] > 2.0 ** -15 * np.abs(q[:, h]).sum(1) * size * 0.125 + 30
        if past == 0:
            far[0] = True
        best = t.argmax(1)
        scale = c.vs[table[0][best // 64], kv_head].astype(np.float64)
        assert np.all((np.abs(got[:, h] - values[kv_head][best]) <= 2.0 ** -20 * 448 * scale[:, None])[far]), h
        tried += far.sum()
    assert tried > 0.5 * heads * new


@pytest.mark.parametrize("new,heads,kv,d", [(2, 4, 2, 64), (50, 4, 2, 64), (90, 4, 2, 128), (650, 64, 2, 32)])
@pytest.mark.parametrize("size", [1.0, 1e3, 3e4, 1e6])
def test_equal_scores_of_any_size_share_a_row(ctx, new, heads, kv, d, size):
    """All keys alike, whatever the values' scales: rows are the average of what they see.  Weights are equal numbers, so what is off is the sums, of 2^-23 an
    addition at most, and values' products."""
    rng = np.random.default_rng(int(size))
    past = 448
    table, lens, starts, pages = S.layout(rng, [new], [past])
    n = int(lens[0])
    k = np.repeat(rng.standard_normal((1, kv, d)).astype(np.float32), n, 0) * np.float32(size)
    v = rng.standard_normal((n, kv, d)).astype(np.float32)
    c = F.Cache(pages, kv, d)
    c.append(k, v, table, lens, np.array([0, n]))
    c.vs *= np.float32(2) ** rng.integers(-9, 9, c.vs.shape).astype(np.float32)
    q = (rng.standard_normal((new, heads, d)) * size).astype(np.float32)
    _, values = c.tokens(table[0], n)
    upto = np.cumsum(values, 1)[:, past:] / np.arange(past + 1, n + 1)[None, :, None]
    want = np.repeat(upto, heads // kv, 0).transpose(1, 0, 2)
    got = T.attend_tree(ctx, c, q, table, lens, starts, chain(new), 1.0)
    assert X.relative(got, want) <= 2.0 ** -20, (X.relative(got, want) * 2 ** 20)


@pytest.mark.parametrize("new,heads,kv,d", [(2, 4, 2, 64), (30, 4, 2, 128), (90, 4, 2, 32)])
@pytest.mark.parametrize("octaves", [24, 31, 34])
def test_many_small_weights_beside_a_large_one(ctx, new, heads, kv, d, octaves):
    """20000 tokens with weights of 2^-octaves, whose values do not cancel: 2^-20 as above, and no more than 2^-32 of the largest share for each of them."""
    rng = np.random.default_rng(octaves)
    past = 20000
    table, lens, starts, pages = S.layout(rng, [new], [past])
    n = int(lens[0])
    k, v = np.zeros((n, kv, d), np.float32), rng.uniform(1, 2, (n, kv, d)).astype(np.float32)
    k[:, :, 0], k[3, :, 0] = -octaves * np.log(2) / 16 / d ** -0.5, 0
    q = np.zeros((new, heads, d), np.float32)
    q[:, :, 0] = 16
    c = F.Cache(pages, kv, d)
    c.append(k, v, table, lens, np.array([0, n]))
    want = X.attention(c, q, table[0], n, d ** -0.5)
    got = T.attend_tree(ctx, c, q, table, lens, starts, chain(new), np.float32(d ** -0.5))
    assert np.all(np.abs(got - want) <= 2 * (2.0 ** -20 + n * 2.0 ** -32))


# ---- precision ----------------------------------------------------------------------------------------
def any_cache(rng, new, past, kv, d):
    """A cache of normally distributed elements, its scales any numbers of a size."""
    table, lens, starts, pages = S.layout(rng, new, past)
    c = F.Cache(pages, kv, d)
    pool = F.encode(rng.standard_normal(4099) * 64)
    c.k[:], c.v[:] = (rng.choice(pool, x.shape) for x in (c.k, c.v))
    for s in (c.ks, c.vs):
        s[:] = rng.uniform(0.7, 1.4, s.shape) / 64
    return c, table, lens, starts


def attention_of_trees(c, q, table, lens, starts, mask, alpha):
    out = np.empty(q.shape)
    group = q.shape[1] // c.heads
    for s, length in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        n, past = b - a, length - (b - a)
        k, v = (torch.from_numpy(t) for t in c.tokens(table[s], int(length)))
        sees = torch.ones((n, int(length)), dtype=torch.bool)
        sees[:, past:] = torch.from_numpy(D.unpack(mask[a:b], n)[:, :n])
        for h in range(q.shape[1]):
            t = torch.from_numpy(q[a:b, h].astype(np.float64)) @ k[h // group].T * alpha
            out[a:b, h] = (torch.softmax(t.masked_fill(~sees, -np.inf), 1) @ v[h // group]).numpy()
    return out


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("new,past,heads,kv", tree_plan.CASES)
def test_attention_in_2_norm(ctx, new, past, heads, kv, d):
    """In every form of items.  (The bound: see test_gpu_fp8_edges.test_values_of_pages_that_differ_in_size.)"""
    rng = np.random.default_rng(sum(new) + d)
    c, table, lens, starts = any_cache(rng, new, past, kv, d)
    q = rng.standard_normal((sum(new), heads, d)).astype(np.float32)
    mask = H.tree_mask(np.concatenate([D.tree(rng, n, 3) for n in new]), starts)
    want = attention_of_trees(c, q, table, lens, starts, mask, d ** -0.5)
    got = T.attend_tree(ctx, c, q, table, lens, starts, mask, np.float32(d ** -0.5))
    assert X.relative(got, want) <= 2.0 ** -20, X.relative(got, want) * 2.0 ** 20


# ---- shares beside the largest that float16 parts take ------------------------------------------------
@pytest.mark.parametrize("low,high", [(-96, -92), (60, 64), (-30, -27), (-96, -91), (3, 7)])
@pytest.mark.parametrize("seqs,new,heads,kv,d,pages", [(60, 3, 8, 4, 64, 16), (60, 3, 8, 4, 128, 16), (32, 50, 8, 8, 64, 16), (32, 32, 32, 8, 128, 24)])
def test_shares_beside_the_largest(ctx, seqs, new, heads, kv, d, pages, low, high):
    """Pages of scale 2^low with scores of 0, then pages of 2^high with a score s at which their shares cross 2^15 in the units that the first ones set (with
    2^9 for their own), s a few steps of fp32 apart from row to row: whether a row changes its units hangs on how sums of s, exponents and units round, and all that
    ask for it have to agree.  A row is the average of two averages; s is off by (3 + d / 8) 2^-23 of itself, as above, and 2^-18 is more than that and 2^-20."""
    assert not tree_plan.form_of([new] * seqs, [64 * pages] * seqs, heads, kv, d)[1]   # (a workgroup goes through all pages of an item)
    rng = np.random.default_rng(high - low)
    c = F.Cache(pages + seqs, kv, d)
    second = np.arange(pages + seqs) >= pages // 2
    c.k[:], c.k[second, ..., 0] = 0, F.encode(1.0)
    c.v[:] = rng.choice(F.encode(rng.standard_normal(4099) * 64), c.v.shape)
    c.ks[:] = 1
    c.vs[:] = np.where(second, 2.0 ** high, 2.0 ** low)[:, None]
    table = np.concatenate([np.tile(np.arange(pages), (seqs, 1)), pages + np.arange(seqs)[:, None]], 1).astype(np.int32)
    lens, starts = np.full(seqs, 64 * pages + new, np.int32), (new * np.arange(seqs + 1)).astype(np.int32)
    target = 15 - (9 + high - low)                                            # of s, a power of two's exponent
    q = np.zeros((seqs * new, heads, d), np.float32)
    steps = np.arange(seqs * new * heads).reshape(seqs * new, heads) % 128 - 64
    q[:, :, 0] = target / np.log2(np.e) * (1 + steps * 2.0 ** -23)
    s = q[:, :, 0].astype(np.float64) * np.log2(np.e)
    assert s.min() < target < s.max()
    values = np.repeat(np.moveaxis(F.decode(c.v[:pages]), 3, 2), heads // kv, 1)   # [pages, heads, tokens, d]
    first, rest = (values[part].mean((0, 2)) * scale for part, scale in ((slice(0, pages // 2), 2.0 ** low), (slice(pages // 2, None), 2.0 ** high)))
    weight = (2.0 ** s / (1 + 2.0 ** s))[:, :, None]
    want = (1 - weight) * first + weight * rest
    got = T.attend_tree(ctx, c, q, table, lens, starts, np.zeros((seqs * new, 2), np.int32), 1.0)
    assert X.relative(got, want) <= 2.0 ** -18, X.relative(got, want) * 2.0 ** 20
