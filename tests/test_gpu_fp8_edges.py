"""The 8-bit serving operators at operands where a definition and a shortcut part: quotients beside a tie, pages of
values that differ in size, scales that are no numbers, scales of every size, more blocks than a launch has threads
for, rows whose factor is no normal number, scores beyond 2^24, more rows than a grid has workgroups for."""
import numpy as np
import pytest
import torch

import fp8_ref as F
import test_gpu_fp8_serving as S
from webdnn_amd import capi
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


# ---- quantisation is a division ------------------------------------------------------------------
def quotients(x, scales, block_rows):
    """e4m3 bytes of the fp32 quotients of finite x and its blocks' scales (numpy divides fp32 numbers with one rounding)."""
    c = np.repeat(np.repeat(scales, block_rows, 0), 128, 1)[:x.shape[0], :x.shape[1]]
    y = np.clip(x / c, np.float32(-448), np.float32(448))
    return torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def beside_ties(rng, rows, cols, block_rows, sizes):
    """Elements whose quotient by their block's scale is a middle between two e4m3 values, or a few fp32 steps from one."""
    top = (rng.uniform(1, 2, (-(-rows // block_rows), -(-cols // 128))) * 448).astype(np.float32) * sizes
    c = np.maximum(top / np.float32(448), np.float32(F.LEAST))
    per = lambda t: np.repeat(np.repeat(t, block_rows, 0), 128, 1)[:rows, :cols]
    ties = np.concatenate([(F.VALUES[:126] + F.VALUES[1:127]) / 2, F.VALUES[:127]])
    x = (rng.choice(ties, (rows, cols)) * per(c).astype(np.float64)).astype(np.float32)
    x = (x.view(np.int32) + np.where(x != 0, rng.integers(-2, 3, (rows, cols)), 0).astype(np.int32)).view(np.float32)
    x = np.minimum(x, per(top)) * np.where(rng.random((rows, cols)) < 0.5, np.float32(-1), np.float32(1))
    x[::block_rows, ::128] = top
    return x


@pytest.mark.parametrize("size", [1.0, 2.0 ** -40, 2.0 ** -41, 2.0 ** -98, 2.0 ** -110, 2.0 ** 60, 2.0 ** 118])
@pytest.mark.parametrize("rows,cols,block_rows", [(40, 1030, 1), (333, 128, 1), (300, 1028, 128), (512, 130, 128)])
def test_quantised_values_are_those_of_the_quotients(ctx, rows, cols, block_rows, size):
    rng = np.random.default_rng(rows + cols)
    x = beside_ties(rng, rows, cols, block_rows, np.float32(size))
    q, c = (t.get_data() for t in H.quantize_fp8(ctx, ctx.move_tensor(x), block_rows))
    want = np.maximum(F.finite_amax(F.block_view(x, block_rows), (1, 3)) / np.float32(448), np.float32(F.LEAST))
    assert np.array_equal(c, want) and F.same_bytes(q, quotients(x, c, block_rows))


@pytest.mark.parametrize("rows,length", [(9, 128), (40, 1030), (7, 4096), (3, 20000)])
def test_a_norms_8_bit_rows_are_the_quotients_of_its_fp32_ones(ctx, rows, length):
    rng = np.random.default_rng(length)
    x = (rng.standard_normal((rows, length)) * 2.0 ** rng.integers(-8, 8, (rows, length))).astype(np.float32)
    y, q, c = ctx.empty_tensor(x.shape), ctx.empty_tensor(x.shape, "float8e4m3fn"), ctx.empty_tensor([rows, -(-length // 128)])
    H.call("wdh_rmsnorm", ctx.move_tensor(x).handle, 0, 0, 0, y.handle, q.handle, c.handle, rows, length, 1e-5)
    assert F.same_bytes(q.get_data(), quotients(y.get_data(), c.get_data(), 1))


# ---- attention over pages whose values differ in size ----------------------------------------------
def sized_pages(rng, new, past, heads, kv, d, large, octaves):
    """Sequences of one call, some pages of which hold values 2^octaves as large as the others', behind keys that no query wants
    (60 nats below the others, weights of 2^-86): (cache, table, lens, starts, q)."""
    table, lens, starts, pages = S.layout(rng, [new], [past])
    n = int(lens[0])
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((new, heads, d)).astype(np.float32)
    k[:, :, 0], q[:, :, 0] = 0, 16
    for page in large:
        at = slice(64 * page, 64 * page + 64)
        k[at, :, 0] = -30 * 0.125 / d ** -0.5
        v[at] *= np.float32(2.0 ** octaves)
    c = F.Cache(pages, kv, d)
    c.append(k, v, table, lens, np.array([0, n]))
    return c, table, lens, starts, q


def attention(c, q, table_row, length, alpha):
    """The last len(q) tokens of one sequence in 64 bits."""
    k, v = (torch.from_numpy(t) for t in c.tokens(table_row, length))
    n, heads, d = q.shape
    past, group = torch.arange(n)[:, None] + length - n, heads // len(k)
    out = np.empty(q.shape)
    for h in range(heads):
        t = torch.from_numpy(q[:, h].astype(np.float64)) @ k[h // group].T * alpha
        out[:, h] = (torch.softmax(t.masked_fill(torch.arange(length) > past, -np.inf), 1) @ v[h // group]).numpy()
    return out


def relative(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("octaves", [0, 16, 20, 30, 40, 60, 82])
@pytest.mark.parametrize("new,heads,kv,d,large", [(1, 4, 2, 64, [0]), (90, 4, 2, 64, [2]), (650, 64, 2, 64, [0]), (650, 64, 2, 64, [3, 7]), (650, 64, 2, 64, [11]),
                                                  (700, 32, 4, 128, [1]), (1300, 64, 2, 32, [0, 9])])
def test_values_of_pages_that_differ_in_size(ctx, new, heads, kv, d, large, octaves):
    """What a row attends to counts in full, however large the values are that it does not attend to.

    2-norm over all results: a score's 3 d / 32 additions of its queries' parts and the roundings of its factor, argument and power
    are some 2^-22.5 of a weight, different for each key (scores here are of size one); sums and second products add less.
    2^-20 is four times that; weights or queries cut to 16 or fewer bits are 2^-17 and more.  (2^82 times as large, the values behind weights of
    2^-86 show in the results.)"""
    rng = np.random.default_rng(octaves)
    past = 640
    c, table, lens, starts, q = sized_pages(rng, new, past, heads, kv, d, large, octaves)
    want = attention(c, q, table[0], int(lens[0]), d ** -0.5)
    got = S.attend(ctx, c, q, table, lens, starts, np.float32(d ** -0.5))
    assert relative(got, want) <= 2.0 ** -20, (relative(got, want) * 2 ** 20)
    assert np.max(np.abs(want)) < 64                                         # (no row rests on a large page)


# ---- scales that are no numbers ----------------------------------------------------------------------
@pytest.mark.parametrize("past,new", [(64, 1), (0, 1), (63, 2), (128, 1), (640, 1)])
def test_an_infinite_key_scale_shows_in_a_page_of_one_key(ctx, past, new):
    """The page's only key lies against the query: its score would be -inf, whose weight is 0, if the scale were multiplied with."""
    rng = np.random.default_rng(past)
    c, table, lens, starts = S.filled(rng, [new], [past], 2, 64)
    n = int(lens[0])
    k, _ = c.tokens(table[0], n)
    q = rng.standard_normal((new, 4, 64)).astype(np.float32)
    q[-1] = -np.repeat(k[:, n - 1], 2, 0)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    c.ks[table[0, (n - 1) // 64], 1] = np.inf
    got = S.attend(ctx, c, q, table, lens, starts, 0.125)
    assert np.isnan(got[-1, 2:]).all()
    assert np.all((np.abs(got - want) <= bound)[:, :2]) and np.all((np.abs(got - want) <= bound)[:-1])


# ---- products of extreme scales ----------------------------------------------------------------------
SHAPES = [(1, 40, 700), (2, 300, 1040), (3, 50, 260), (20, 200, 12000), (40, 300, 1024), (100, 900, 2050), (300, 700, 4096), (700, 2000, 130), (1500, 2000, 144),
          (8192, 4096, 200)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("a_octave,w_octave", [(70, -90), (-70, 90), (-140, 110), (127, -149), (-100, -24), (-62, -62), (60, 60), (120, 0), (-100, -100)])
def test_scales_of_any_size_with_a_normal_product(ctx, m, n, k, a_octave, w_octave):
    """Every third block has extreme scales; their product is 2^-126 to 2^122, or 0 as for blocks of zeros, whose scales are 2^-100 both.
    Half the rows have one element in each of these blocks and nothing else: small terms count for themselves.  One row is zeros."""
    rng = np.random.default_rng(m + n)
    kb, nb = -(-k // 128), -(-n // 128)
    odd = np.arange(kb) % 3 == 0                                             # (the others have scales of size one)
    a, w = S.bytes_of(rng, (m, k)), S.bytes_of(rng, (n, k))
    sa, sw = (rng.uniform(1, 2, s).astype(np.float32) for s in ((m, kb), (nb, kb)))
    sa[:, odd] *= np.float32(2.0 ** a_octave)
    sw[:, odd] *= np.float32(2.0 ** w_octave)
    if a_octave < -126 or w_octave < -126:                                   # (subnormal ones have few bits)
        sa[:, odd], sw[:, odd] = np.float32(2.0 ** a_octave), np.float32(2.0 ** w_octave)
    alone = rng.random(m) < 0.5
    in_odd = np.repeat(odd, 128)[:k]
    a[np.ix_(alone, ~in_odd)] = 0
    a[np.ix_(alone, np.arange(k) % 128 != 5)] = 0
    if a_octave + w_octave > 100:
        a[:, in_odd] &= 0x83                                                 # subnormal values: at most 3 * 2^-9
        w[:, in_odd] &= 0x83
    if a_octave + w_octave == -200:
        a[:, in_odd] &= 0x80
        w[:, in_odd] &= 0x80
    a[0] = 0x80
    want, size = F.product(a, sa, w, sw)
    y = H.matmul_fp8(ctx, *(ctx.move_tensor(t) for t in (a, sa, w, sw))).get_data().astype(np.float64)
    assert np.array_equal(y[0], np.zeros(n))
    # a block's sum (of one product: nothing), its scales' product, the product with it, the sum of blocks; at most 2^-23 of the sizes' sum each
    bound = np.where(alone, 3 + kb, 128 + 3 + kb)[:, None] * 2 * E * size + kb * 2.0 ** -149
    assert size.max() < 3e38 and np.all(np.abs(y - want) <= bound), float(np.max(np.abs(y - want) - bound))


@pytest.mark.parametrize("m", [1, 3, 300])
def test_scales_that_are_no_numbers_reach_their_rows_and_columns(ctx, m):
    rng = np.random.default_rng(m)
    n, k = 300, 260
    a, w = S.bytes_of(rng, (m, k)), S.bytes_of(rng, (n, k))
    sa, sw = np.ones((m, 3), np.float32), np.ones((3, 3), np.float32)
    sa[m - 1, 1], sw[2, 0], sw[1, 2] = np.nan, np.inf, 0
    y = H.matmul_fp8(ctx, *(ctx.move_tensor(t) for t in (a, sa, w, sw))).get_data()
    bad = np.zeros((m, n), bool)
    bad[m - 1], bad[:, 256:] = True, True
    assert np.array_equal(~np.isfinite(y), bad) and np.isnan(y[m - 1]).all()


# ---- limits --------------------------------------------------------------------------------------------
def test_blocks_beyond_a_launch_are_refused(ctx):
    """A launch has fewer than 2^32 threads; a block of 1 x 128 takes eight."""
    for rows, cols in ((1 << 29, 1), (1 << 28, 129), ((1 << 29) - 31, 128)):
        with pytest.raises(capi.HipError) as err:
            H.call("wdh_quantize_fp8", 1, 1, 1, rows, cols, 1)
        assert err.value.code == -2 and "too many blocks" in str(err.value)


def test_as_many_blocks_as_a_launch_has(ctx):
    rows, n = (1 << 29) - 32, 1000
    x, q, c = ctx.empty_tensor([rows, 1]), ctx.empty_tensor([rows, 1], "float8e4m3fn"), ctx.empty_tensor([rows, 1])
    some = np.random.default_rng(1).standard_normal((n, 1)).astype(np.float32)
    ends = (0, rows - n)
    for at in ends:
        H.call("wdh_write", x.handle, 4 * at, some.ctypes.data, some.nbytes)
    H.quantize_fp8(ctx, x, 1, out=(q, c))
    for at in ends:
        byte, scale = np.empty((n, 1), np.uint8), np.empty((n, 1), np.float32)
        H.call("wdh_read", q.handle, at, byte.ctypes.data, n)
        H.call("wdh_read", c.handle, 4 * at, scale.ctypes.data, 4 * n)
        assert np.array_equal(scale, np.abs(some) / np.float32(448)) and F.same_bytes(byte, quotients(some, scale, 1))
    for t in (x, q, c):
        t.dispose()
    ctx.sync()
    capi.call("wdh_trim", 0)


# ---- rows whose factor is no normal number ---------------------------------------------------------------
@pytest.mark.parametrize("length", [200, 700, 3000, 9000, 20000])
@pytest.mark.parametrize("size", [1e-45, 1e-42, 1e-39, 1e-38, 1e-35, 1e30, 5e36, 5e37, 3e38])
def test_norm_of_the_least_and_largest_rows(ctx, length, size):
    """1 / sqrt(mean) of such rows is beyond fp32's numbers, or among its subnormal ones."""
    rng = np.random.default_rng(length)
    x = (rng.standard_normal((3, length)).clip(-1.1, 1.1) * size).astype(np.float32)
    x[:, 0] = np.float32(size)
    g = rng.uniform(0.5, 1.5, length).astype(np.float32)
    want = F.rms(x.astype(np.float64), g.astype(np.float64), 0.0)
    y = H.rms_normalization(ctx, ctx.move_tensor(x), ctx.move_tensor(g), epsilon=0.0).get_data()
    assert np.all(np.abs(y - want) <= 3.01 * E * np.abs(want) + 2.0 ** -149)


# ---- scores beyond 2^24 ------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [1e2, 3e3, 1e4, 1e5, 1e7, 1e9, 1e14])
@pytest.mark.parametrize("new,past,heads,kv,d", [(1, 900, 8, 2, 64), (60, 100, 4, 2, 128), (1, 3000, 2, 1, 128), (650, 100, 64, 2, 64), (700, 0, 32, 4, 128)])
@pytest.mark.parametrize("alpha", [1.0, -0.125])
def test_scores_of_any_size(ctx, new, past, heads, kv, d, size, alpha):
    """Where neighbouring fp32 numbers are further apart than the powers of two that weights are, rows rest on their largest score: the others
    are left far behind (rows whose two largest scores are not further apart than their errors are left out)."""
    rng = np.random.default_rng(new)
    table, lens, starts, pages = S.layout(rng, [new], [past])
    n = int(lens[0])
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in range(2))
    c = F.Cache(pages, kv, d)
    c.append(k * np.float32(size), v, table, lens, np.array([0, n]))
    c.ks *= rng.uniform(0.5, 1, c.ks.shape).astype(np.float32)               # (append writes powers of two, but any number will do)
    q = (rng.standard_normal((new, heads, d)) * size).astype(np.float32)
    keys, values = c.tokens(table[0], n)
    got = S.attend(ctx, c, q, table, lens, starts, alpha)
    tried = 0
    for h in range(heads):
        t = q[:, h].astype(np.float64) @ keys[h // (heads // kv)].T * alpha
        t[np.arange(n) > np.arange(new)[:, None] + past] = -np.inf
        order = np.sort(t, 1)
        far = np.ones(new, bool) if n == 1 else order[:, -1] - order[:, -2] > 2.0 ** -15 * np.abs(q[:, h]).sum(1) * size * abs(alpha) + 30
        if past == 0:
            far[0] = True
        want = values[h // (heads // kv)][t.argmax(1)]
        assert np.all(np.abs(got[:, h] - want)[far] <= 2.0 ** -20 * np.abs(values).max()), (h, got[:, h][far])
        tried += far.sum()
    assert tried > 0.7 * heads * new


# ---- more rows than a grid has workgroups for --------------------------------------------------------------
@pytest.mark.parametrize("rows,length", [(4200003, 5), (1050001, 300)])
def test_norm_of_millions_of_rows(ctx, rows, length):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((1000, length)).astype(np.float32)
    dx = ctx.empty_tensor([rows, length])
    ends = (0, rows // 2, rows - 1000)
    for at in ends:
        H.call("wdh_write", dx.handle, 4 * at * length, x.ctypes.data, x.nbytes)
    y = H.rms_normalization(ctx, dx)
    want = F.rms(x.astype(np.float64), None, 1e-5)
    got = np.empty_like(x)
    for at in ends:
        H.call("wdh_read", y.handle, 4 * at * length, got.ctypes.data, got.nbytes)
        assert np.all(np.abs(got - want) <= 3.01 * E * np.abs(want))
    for t in (dx, y):
        t.dispose()
    ctx.sync()
    capi.call("wdh_trim", 0)


@pytest.mark.parametrize("m,n,k", [(1, 4194400, 17), (2, 4200001, 16), (2200001, 3, 17), (1100003, 9, 48), (1100001, 17, 40), (300001, 200, 130), (7, 5000001, 16)])
def test_products_of_millions_of_rows(ctx, m, n, k):
    rng = np.random.default_rng(m + n)
    a, w = S.bytes_of(rng, (m, k)), S.bytes_of(rng, (n, k))
    kb = -(-k // 128)
    sa, sw = (rng.uniform(0.5, 1, s).astype(np.float32) for s in ((m, kb), (-(-n // 128), kb)))
    y = H.matmul_fp8(ctx, *(ctx.move_tensor(t) for t in (a, sa, w, sw))).get_data()
    for begin in range(0, max(m, n), 500000):                                # (the oracle's 64-bit copies a piece at a time)
        i, j = (slice(begin, begin + 500000) if side > 1000 else slice(0, side) for side in (m, n))
        columns = slice(j.start // 128, -(-min(j.stop, n) // 128))
        lead = j.start % 128
        w_piece, sw_piece = w[j.start - lead:j.stop], sw[columns]
        want, size = (t[:, lead:] for t in F.product(a[i], sa[i], w_piece, sw_piece))
        assert np.all(np.abs(y[i, j] - want) <= (128 + 2 + kb) * 2 * E * size)
