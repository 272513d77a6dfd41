"""The 8-bit serving operators on the GPU against their definitions in 64 bits (fp8_ref): root-mean-square norm, quantisation in
blocks, e4m3 products, the paged cache and attention over it; their refusals; and a run of them together, recorded and not.

In the reference's terms they are chains of src/descriptor_runner/operators/cpu/operators/standard/{binary7,reduce,unary,matmul,softmax}.ts.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

import fp8_ref as F
from webdnn_amd import capi
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def bytes_of(rng, shape):
    """e4m3 bytes of every size, none of them NaN."""
    b = rng.integers(0, 127, shape).astype(np.uint8)
    return b | (rng.integers(0, 2, shape).astype(np.uint8) << 7)


# ---- norm -------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,length", [(1, 1), (3, 127), (5, 128), (6, 129), (2, 256), (9, 257), (3, 512), (4, 1000), (7, 1024), (3, 1030), (2, 2049),
                                         (1, 4096), (3, 4099), (2, 8191), (2, 8193), (1, 20001), (0, 7), (4, 0)])
@pytest.mark.parametrize("skip,scaled", [(True, True), (False, False)])
def test_norm(ctx, rows, length, skip, scaled):
    rng = np.random.default_rng(rows * 100003 + length)
    x, r = (rng.standard_normal((rows, length)).astype(np.float32) * np.exp(rng.standard_normal(length)).astype(np.float32) for _ in range(2))
    g = rng.uniform(-2, 2, length).astype(np.float32) if scaled else None
    s = (x + r) if skip else x
    want = F.rms(s.astype(np.float64), None if g is None else g.astype(np.float64), 1e-5) if length else s
    dx, dr, dg = ctx.move_tensor(x), ctx.move_tensor(r) if skip else None, ctx.move_tensor(g) if scaled else None
    got = H.rms_normalization(ctx, dx, dg, dr)
    total, y = got if skip else (None, got)
    y = y.get_data()
    # 1/sqrt rounded once (its argument is in 64 bits), and a rounding for each of two products
    assert np.all(np.abs(y - want) <= 3.01 * E * np.abs(want) + 2.0 ** -149)
    got = H.rms_normalization_fp8(ctx, dx, dg, dr)
    q, c = (t.get_data() for t in got[-2:])
    F.check_quantized(q, c, want, 1, 3.01 * E)
    for t in (total, got[0]) if skip else ():
        assert np.array_equal(t.get_data(), s)


def test_norm_updates_the_stream_in_place_and_gives_both_forms(ctx):
    rng = np.random.default_rng(1)
    for length in (300, 9000):
        x, r = (rng.standard_normal((5, length)).astype(np.float32) for _ in range(2))
        want = F.rms((x + r).astype(np.float64), None, 1e-6)
        for into in (0, 1):
            dx, dr = ctx.move_tensor(x), ctx.move_tensor(r)
            place = (dx, dr)[into]
            y, q, c = ctx.empty_tensor(x.shape), ctx.empty_tensor(x.shape, "float8e4m3fn"), ctx.empty_tensor([5, -(-length // 128)])
            H.call("wdh_rmsnorm", dx.handle, dr.handle, 0, place.handle, y.handle, q.handle, c.handle, 5, length, 1e-6)
            assert np.array_equal(place.get_data(), x + r) and np.array_equal((dr, dx)[into].get_data(), (r, x)[into])
            assert np.all(np.abs(y.get_data() - want) <= 3.01 * E * np.abs(want))
            F.check_quantized(q.get_data(), c.get_data(), want, 1, 3.01 * E)


@pytest.mark.parametrize("length", [200, 3000])
def test_norm_of_extreme_rows(ctx, length):
    """Zeros, squares beyond and below fp32's range, and rows with an infinity or a NaN."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, length)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e25)
    x[2] *= np.float32(1e-30)
    x[3, 7], x[4, 9] = np.inf, np.nan
    dx = ctx.move_tensor(x)
    y = H.rms_normalization(ctx, dx, epsilon=0.0).get_data()
    q, c = (t.get_data() for t in H.rms_normalization_fp8(ctx, dx, epsilon=1e-5))
    for i in (1, 2, 5):
        want = F.rms(x[i:i + 1].astype(np.float64), None, 0.0)
        assert np.all(np.abs(y[i] - want) <= 3.01 * E * np.abs(want)), i
    assert np.isnan(y[0]).all() and np.isnan(y[4]).all()                    # 0 / 0, and NaN
    assert np.isnan(y[3, 7]) and np.all(np.delete(y[3], 7) == 0)            # x / inf
    assert np.all(q[0] == 0) and np.all(c[0] == np.float32(F.LEAST)) and np.all((q[4] & 127) == 127)


# ---- quantisation --------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 127), (3, 128), (129, 130), (300, 257), (1, 4100), (65, 1030), (128, 384), (0, 9), (9, 0)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(ctx, rows, cols, block_rows):
    rng = np.random.default_rng(rows + 1000 * cols)
    x = (rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-20, 20, (rows, 1))).astype(np.float32)
    q, c = (t.get_data() for t in H.quantize_fp8(ctx, ctx.move_tensor(x), block_rows))
    F.check_quantized(q, c, x.astype(np.float64), block_rows, 0.0)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(ctx, block_rows):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((256, 384)).astype(np.float32)
    x[0, 3], x[0, 130], x[130, 260], x[130, 300] = np.inf, -np.inf, np.nan, np.float32(3.4e38)
    x[128:, :128] = 0
    x[128:, 128:256] *= np.float32(1e-36)
    x[128:, 200] = np.float32(1e-45)
    q, c = (t.get_data() for t in H.quantize_fp8(ctx, ctx.move_tensor(x), block_rows))
    F.check_quantized(q, c, x.astype(np.float64), block_rows, 0.0)


# ---- products ------------------------------------------------------------------------------------
def check_product(ctx, rng, m, n, k, bias=False, residual=False, relu=False):
    a, w = bytes_of(rng, (m, k)), bytes_of(rng, (n, k))
    kb = -(-k // 128)
    sa = (2.0 ** rng.integers(-12, 4, (m, kb)) * rng.uniform(0.5, 1, (m, kb))).astype(np.float32)
    sw = (2.0 ** rng.integers(-12, 4, (-(-n // 128), kb)) * rng.uniform(0.5, 1, (-(-n // 128), kb))).astype(np.float32)
    want, size = F.product(a, sa, w, sw)
    # a block's sum: 128 additions; its scale: two roundings; the sum of blocks in any order; at most 2^-23 of the sizes' sum each
    bound = (128 + 2 + kb) * 2 * E * size
    b = rng.standard_normal(n).astype(np.float32) * np.float32(100) if bias else None
    r = rng.standard_normal((m, n)).astype(np.float32) * np.float32(100) if residual else None
    for t in (b, r):
        if t is not None:
            want = want + t.astype(np.float64)
            bound = bound + E * (np.abs(want) + bound)
    if relu:
        want = np.maximum(want, 0)
    up = lambda t: None if t is None else ctx.move_tensor(t)
    y = H.matmul_fp8(ctx, up(a), up(sa), up(w), up(sw), up(b), up(r), "relu" if relu else None).get_data()
    assert y.shape == (m, n) and np.all(np.abs(y - want) <= bound), float(np.max(np.abs(y - want) - bound))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 129, 200])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 130), (128, 256), (129, 2050), (300, 48), (257, 1040), (64, 4096)])
def test_product(ctx, m, n, k):
    check_product(ctx, np.random.default_rng(m * 7919 + n * 31 + k), m, n, k, bias=m % 2 == 0, residual=n % 2 == 1, relu=m == 33)


@pytest.mark.parametrize("m,n,k", [(513, 384, 1024), (300, 1000, 520), (1025, 260, 272), (256, 512, 2048), (777, 333, 129), (2048, 1024, 640)])
def test_larger_products(ctx, m, n, k):
    check_product(ctx, np.random.default_rng(m + n + k), m, n, k, bias=True, residual=True)


def test_products_without_rows_or_inner_dimension(ctx):
    e8 = lambda *s: ctx.empty_tensor(s, "float8e4m3fn")
    y = H.matmul_fp8(ctx, e8(0, 200), ctx.empty_tensor([0, 2]), e8(5, 200), ctx.empty_tensor([1, 2]))
    assert y.get_data().shape == (0, 5)
    b, r = np.arange(5, dtype=np.float32) - 2, np.ones((3, 5), np.float32)
    y = H.matmul_fp8(ctx, e8(3, 0), ctx.empty_tensor([3, 0]), e8(5, 0), ctx.empty_tensor([1, 0]), ctx.move_tensor(b), ctx.move_tensor(r), "relu")
    assert np.array_equal(y.get_data(), np.maximum(b + r, 0))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_product_takes_nan_and_residual_in_place(ctx, m):
    """A NaN of A reaches its row and no other, one of W its column; the residual may be the result's own buffer."""
    rng = np.random.default_rng(11)
    n, k = 150, 272
    a, w = bytes_of(rng, (m, k)), bytes_of(rng, (n, k))
    a[1, 200], w[140, 5] = 0x7f, 0xff
    sa, sw = np.full((m, 3), 0.01, np.float32), np.full((2, 3), 0.02, np.float32)
    r = rng.standard_normal((m, n)).astype(np.float32)
    y = ctx.move_tensor(r)
    H.matmul_fp8(ctx, ctx.move_tensor(a), ctx.move_tensor(sa), ctx.move_tensor(w), ctx.move_tensor(sw), residual=y, out=y)
    got = y.get_data()
    nan = np.zeros((m, n), bool)
    nan[1], nan[:, 140] = True, True
    assert np.array_equal(np.isnan(got), nan)
    want, size = F.product(a, sa, w, sw)
    bound = (128 + 2 + 3) * 2 * E * size + E * (np.abs(want + r) + 1)
    assert np.all(np.abs(got - (want + r))[~nan] <= bound[~nan])


# ---- the cache -----------------------------------------------------------------------------------
def layout(rng, new, past, extra=2):
    """table, lens, starts of sequences on pages in random order; unused entries name no page."""
    lens = np.array(new) + np.array(past)
    count = -(-lens // 64)
    order = rng.permutation(int(count.sum()) + extra)
    table = np.full((len(new), max(1, int(count.max()))), -7, np.int32)
    at = 0
    for s, c in enumerate(count):
        table[s, :c] = order[at:at + c]
        at += c
    return table, lens.astype(np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32), len(order)


def on_device(ctx, c):
    return H.KvCache(ctx, *(ctx.move_tensor(t) for t in (c.k, c.ks, c.v, c.vs)))


def check_cache(device, c):
    for name, got, want in (("k", device.k, c.k), ("v", device.v, c.v)):
        assert F.same_bytes(got.get_data(), want), name
    for name, got, want in (("k", device.k_scales, c.ks), ("v", device.v_scales, c.vs)):
        assert np.array_equal(got.get_data(), want, equal_nan=True), name


MIXES = [([1], [0]), ([1], [63]), ([1], [64]), ([3, 1, 2], [0, 62, 200]), ([130, 1, 64, 5], [0, 0, 64, 63]), ([1] * 70, list(range(0, 140, 2))),
         ([17, 300], [1, 129])]


@pytest.mark.parametrize("heads,d", [(1, 32), (3, 64), (2, 128)])
@pytest.mark.parametrize("new,past", MIXES)
def test_append(ctx, heads, d, new, past):
    """Two calls, the second with values eight times as large: scales grow, earlier tokens are rounded again."""
    rng = np.random.default_rng(sum(new) * 131 + d)
    table, lens, starts, pages = layout(rng, new, past)
    c = F.Cache(pages, heads, d)
    device = on_device(ctx, c)
    begin = np.concatenate([[0], np.cumsum(past)]).astype(np.int32)
    for which, (ls, st, size) in enumerate([(np.array(past, np.int32), begin, 1.0), (lens, starts, 8.0)]):
        n = int(st[-1])
        k, v = (rng.standard_normal((n, heads, d)).astype(np.float32) * np.float32(size) for _ in range(2))
        if n > 2:
            k[n // 2, :, 3], v[n // 3, 0, 1] = np.inf, np.nan
            v[n // 2] *= np.float32(1e-3)
        wide = np.zeros((n, 2 * heads * d + 12), np.float32)             # both in one projection's rows, after four others
        wide[:, 4:4 + heads * d], wide[:, 8 + heads * d:8 + 2 * heads * d] = k.reshape(n, heads * d), v.reshape(n, heads * d)
        H.cache_append(ctx, device, *[ctx.move_tensor(wide)] * 2, ctx.move_tensor(table), ctx.move_tensor(ls), ctx.move_tensor(st),
                       k_column=4, v_column=8 + heads * d)
        c.append(k, v, table, ls, st)
        check_cache(device, c)


def test_append_leaves_out_what_does_not_fit(ctx):
    """Pages outside the cache, sequences with more rows than tokens, than the table holds, or than the call has: nothing of them is written."""
    rng = np.random.default_rng(3)
    heads, d = 2, 64
    table = np.array([[0, 99], [-1, 1], [2, 3], [4, 5], [6, 7]], np.int32)
    starts = np.array([0, 70, 140, 150, 160, 500], np.int32)
    lens = np.array([70, 70, 5, 300, 340], np.int32)
    c = F.Cache(8, heads, d)
    device = on_device(ctx, c)
    k, v = (rng.standard_normal((200, heads, d)).astype(np.float32) for _ in range(2))
    H.cache_append(ctx, device, ctx.move_tensor(k.reshape(200, -1)), ctx.move_tensor(v.reshape(200, -1)), ctx.move_tensor(table),
                   ctx.move_tensor(lens), ctx.move_tensor(starts))
    c.append(k[:64], v[:64], table[:1], [64], [0, 64])                   # the first page of the first sequence
    whole = F.Cache(8, heads, d)
    whole.append(k[134:140], v[134:140], np.array([[1]]), [6], [0, 6])   # and the second of the second
    for a in ("k", "v", "ks", "vs"):
        getattr(c, a)[1] = getattr(whole, a)[1]
    check_cache(device, c)


def filled(rng, new, past, heads, d, extra=2):
    """A cache that holds the sequences' tokens, everything else being NaN."""
    table, lens, starts, pages = layout(rng, new, past, extra)
    c = F.Cache(pages, heads, d)
    all_starts = np.concatenate([[0], np.cumsum(lens)])
    k, v = (rng.standard_normal((int(all_starts[-1]), heads, d)).astype(np.float32) for _ in range(2))
    c.append(k, v, table, lens, all_starts)
    return c, table, lens, starts


def attend(ctx, c, q, table, lens, starts, alpha, out=None, wide=0):
    n, heads, d = q.shape
    rows = np.full((n, heads * d + 2 * wide), np.nan, np.float32)
    rows[:, wide:wide + heads * d] = q.reshape(n, -1)
    y = H.cache_attention(ctx, on_device(ctx, c), ctx.move_tensor(rows), heads, alpha, ctx.move_tensor(table), ctx.move_tensor(lens),
                          ctx.move_tensor(starts), q_column=wide, out=out)
    return y.get_data().reshape(n, heads, d)


@pytest.mark.parametrize("heads,kv,d", [(1, 1, 32), (8, 1, 64), (6, 2, 128), (4, 4, 128), (40, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [0, 63, 500]), ([3, 1, 2], [61, 64, 700]), ([100, 1, 65, 7], [0, 130, 64, 1000]), ([1], [3000])])
def test_attention(ctx, heads, kv, d, new, past):
    rng = np.random.default_rng(heads * 1009 + sum(past) + d)
    c, table, lens, starts = filled(rng, new, past, kv, d)
    q = rng.standard_normal((int(starts[-1]), heads, d)).astype(np.float32)
    alpha = np.float32(d ** -0.5)
    want, bound = c.attention(q, table, lens, starts, float(alpha))
    got = attend(ctx, c, q, table, lens, starts, alpha, wide=4 * (len(new) % 2))
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))


def test_attention_with_sharp_scores(ctx):
    """Scores of hundreds: one key takes all; equal scores share."""
    rng = np.random.default_rng(8)
    c, table, lens, starts = filled(rng, [2, 90], [400, 0], 2, 64)
    q = rng.standard_normal((92, 4, 64)).astype(np.float32) * np.float32(50)
    q[3] = 0
    want, bound = c.attention(q, table, lens, starts, 1.0)
    got = attend(ctx, c, q, table, lens, starts, 1.0)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("new", [[90], [200]])
def test_nan_behind_a_row_does_not_reach_it(ctx, new):
    """Tokens of the same prompt whose keys or values hold NaN: rows before them are what they are without."""
    rng = np.random.default_rng(9)
    kv, d, heads = 2, 64, 4
    c, table, lens, starts = filled(rng, new, [30], kv, d)
    q = rng.standard_normal((new[0], heads, d)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    hit = lens[0] - 20                                                    # a token in the last page but for its tail
    page, slot = table[0, hit // 64], hit % 64
    c.v[page, 0, 5, slot] = 0x7f
    c.k[page, 1, slot, 9] = 0xff
    got = attend(ctx, c, q, table, lens, starts, 0.125)
    row = hit - 30
    assert np.all(np.abs(got - want)[:row] <= bound[:row])
    assert np.isnan(got[row:, :2, 5]).all() and np.isnan(got[row:, 2:]).all()
    keep = np.delete(np.arange(d), 5)
    assert np.all(np.abs(got - want)[row:, :2][..., keep] <= bound[row:, :2][..., keep])


def test_pages_outside_the_cache_make_their_rows_nan(ctx):
    rng = np.random.default_rng(10)
    c, table, lens, starts = filled(rng, [1, 70, 1], [200, 60, 10], 1, 64)
    q = rng.standard_normal((72, 2, 64)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    table[0, 1], table[1, 1] = 1 << 30, -1
    got = attend(ctx, c, q, table, lens, starts, 0.125)
    assert np.isnan(got[0]).all()
    assert np.all(np.abs(got - want)[1:5] <= bound[1:5]) and np.isnan(got[5:71]).all()   # positions 60..63 see the first page only
    assert np.all(np.abs(got - want)[71] <= bound[71])


def test_rows_of_no_sequence_stay_as_they_are(ctx):
    """Padding behind the last sequence, sequences without rows, with more rows than tokens and beyond the table."""
    rng = np.random.default_rng(12)
    c, table, lens, starts = filled(rng, [1, 4, 2, 3], [70, 0, 9, 64], 2, 32)
    starts = np.concatenate([starts, [starts[-1]]]).astype(np.int32)      # a fifth one: no rows, no tokens
    table, lens = np.concatenate([table, table[:1]]), np.append(lens, 0).astype(np.int32)
    q = rng.standard_normal((16, 4, 32)).astype(np.float32)
    want, bound = c.attention(q[:10], table, lens, starts, 0.2)
    lens[1], lens[3] = 3, 1000
    old = np.full((16, 4 * 32), 7.5, np.float32)
    got = attend(ctx, c, q, table, lens, starts, 0.2, out=ctx.move_tensor(old))
    for a, b in ((0, 1), (5, 7)):
        assert np.all(np.abs(got[a:b] - want[a:b]) <= bound[a:b])
    for a, b in ((1, 5), (7, 16)):
        assert np.all(got[a:b] == 7.5)


# ---- refusals -----------------------------------------------------------------------------------
def test_refusals(ctx):
    f, i, e = lambda *s: ctx.empty_tensor(s), lambda *s: ctx.empty_tensor(s, "int32"), lambda *s: ctx.empty_tensor(s, "float8e4m3fn")
    x = f(4, 200)
    with pytest.raises(H.OperatorError):
        H.rms_normalization(ctx, x, f(199))
    with pytest.raises(H.OperatorError):
        H.rms_normalization(ctx, x, None, f(200))
    with pytest.raises(H.OperatorError):
        H.rms_normalization(ctx, i(4, 200))
    with pytest.raises(H.OperatorError):
        H.rms_normalization_fp8(ctx, x, out=(None, e(4, 200), f(4, 1)))
    with pytest.raises(H.OperatorError):
        H.quantize_fp8(ctx, x, 64)
    with pytest.raises(H.OperatorError):
        H.quantize_fp8(ctx, e(4, 200))
    a, sa, w, sw = e(4, 200), f(4, 2), e(300, 200), f(3, 2)
    for bad in ((x, sa, w, sw), (a, f(4, 1), w, sw), (a, sa, e(300, 199), sw), (a, sa, w, f(2, 2)), (a, sa, w, sa)):
        with pytest.raises(H.OperatorError):
            H.matmul_fp8(ctx, *bad)
    with pytest.raises(H.OperatorError):
        H.matmul_fp8(ctx, a, sa, w, sw, bias=f(4))
    with pytest.raises(H.OperatorError):
        H.matmul_fp8(ctx, a, sa, w, sw, residual=f(300))

    def refused(name, *args):
        with pytest.raises(capi.HipError) as err:
            H.call(name, *args)
        assert err.value.code == -2, err.value

    y, q, c = f(4, 200), e(4, 200), f(4, 2)
    h = lambda t: t.handle
    refused("wdh_rmsnorm", h(x), 0, 0, 0, 0, 0, 0, 4, 200, 1e-5)                 # no result
    refused("wdh_rmsnorm", h(x), 0, 0, 0, 0, h(q), 0, 4, 200, 1e-5)              # Q without scales
    refused("wdh_rmsnorm", h(x), 0, 0, 0, h(x), 0, 0, 4, 200, 1e-5)              # Y is X
    refused("wdh_rmsnorm", h(x), 0, 0, h(y), h(y), 0, 0, 4, 200, 1e-5)           # Y is Sum
    refused("wdh_rmsnorm", h(x), 0, 0, 0, h(y), 0, 0, 5, 200, 1e-5)              # too small
    refused("wdh_rmsnorm", h(x), 0, 0, 0, h(y), 0, 0, -1, 200, 1e-5)
    refused("wdh_rmsnorm", h(x), 0, 0, 0, h(y), 0, 0, 4, 200, float("nan"))
    refused("wdh_rmsnorm", h(x), 0, 0, 0, h(y), 0, 0, 1 << 62, 200, 1e-5)
    refused("wdh_quantize_fp8", h(x), h(x), h(c), 4, 200, 1)
    refused("wdh_quantize_fp8", h(x), h(q), h(c), 4, 200, 2)
    refused("wdh_quantize_fp8", h(x), h(q), h(c), 4, 300, 1)
    refused("wdh_gemm_fp8", h(a), h(sa), h(w), h(sw), 0, h(f(4, 299)), 4, 300, 200, 0, 0)
    refused("wdh_gemm_fp8", h(a), h(sa), h(w), h(sw), 0, h(f(4, 300)), 4, 300, 200, 2, 0)
    refused("wdh_gemm_fp8", h(a), h(sa), h(w), h(sw), 0, h(w), 4, 300, 200, 0, 0)
    refused("wdh_gemm_fp8", h(a), 999999, h(w), h(sw), 0, h(f(4, 300)), 4, 300, 200, 0, 0)

    cache = H.KvCache.empty(ctx, 4, 2, 64)
    table, lens, starts = i(3, 2), i(3), i(4)
    with pytest.raises(H.OperatorError):
        H.KvCache(ctx, e(4, 2, 64, 32), cache.k_scales, e(4, 2, 64, 32), cache.v_scales)   # (values are [d][token])
    with pytest.raises(H.OperatorError):
        H.cache_append(ctx, cache, f(5, 128), f(4, 128), table, lens, starts)
    with pytest.raises(H.OperatorError):
        H.cache_append(ctx, cache, f(5, 128), f(5, 128), table, lens, i(3))
    with pytest.raises(H.OperatorError):
        H.cache_append(ctx, cache, f(5, 128), f(5, 128), table, lens, starts, v_column=1)
    with pytest.raises(H.OperatorError):
        H.cache_attention(ctx, cache, f(5, 192), 3, 1.0, table, lens, starts)
    with pytest.raises(H.OperatorError):
        H.cache_attention(ctx, cache, f(5, 256), 4, 1.0, f(3, 2), lens, starts)
    with pytest.raises(H.HipError):                                             # rows that are not whole 16-byte pieces
        H.cache_attention(ctx, cache, f(5, 257), 4, 1.0, table, lens, starts)
    with pytest.raises(H.HipError):
        H.cache_append(ctx, cache, f(5, 132), f(5, 132), table, lens, starts, k_column=2)
    kv = [h(t) for t in (cache.k, cache.k_scales, cache.v, cache.v_scales, table, lens, starts)]
    k, qq, yy = f(5, 128), f(5, 256), f(5, 256)
    refused("wdh_cache_append", h(k), 0, 128, h(k), 0, 128, *kv, 3, 6, 2, 64, 4, 2)     # more tokens than rows
    refused("wdh_cache_append", h(k), 0, 127, h(k), 0, 128, *kv, 3, 5, 2, 64, 4, 2)     # rows that overlap
    refused("wdh_cache_append", h(k), 0, 128, h(k), 0, 128, *kv, 3, 5, 2, 48, 4, 2)     # head dimension
    refused("wdh_cache_append", h(k), 0, 128, h(k), 0, 128, *kv, 3, 5, 2, 64, 5, 2)     # more pages than the cache holds
    refused("wdh_cache_append", h(k), 0, 128, h(k), 0, 128, *kv, 4, 5, 2, 64, 4, 2)     # more sequences than tables
    refused("wdh_cache_append", h(k), 0, 128, h(k), 0, 128, kv[0], kv[1], kv[0], *kv[3:], 3, 5, 2, 64, 4, 2)
    refused("wdh_cache_attention", h(qq), 0, 256, *kv, h(yy), 3, 5, 4, 2, 64, 4, 3, 1.0)
    refused("wdh_cache_attention", h(qq), 0, 256, *kv, h(yy), 3, 5, 5, 2, 64, 4, 2, 1.0)
    refused("wdh_cache_attention", h(qq), 0, 256, *kv, h(qq), 3, 5, 4, 2, 64, 4, 2, 1.0)
    refused("wdh_cache_attention", h(qq), -4, 256, *kv, h(yy), 3, 5, 4, 2, 64, 4, 2, 1.0)
    refused("wdh_cache_attention", h(qq), 0, 256, *kv, h(yy), 3, 5, 4, 2, 64, -1, 2, 1.0)
    for op in ("Relu", "Exp"):                                                  # the fp32 operators do not take e4m3 tensors
        with pytest.raises((H.OperatorError, H.HipError)):
            H.unary(ctx, op, a)
    with pytest.raises((H.OperatorError, H.HipError)):
        H.gemm(ctx, a, w, trans_b=1)


def test_torch_sees_the_same_memory():
    """In a process of its own: torch has to bring the HIP runtime up before this library does."""
    code = """
import numpy as np, torch
torch.zeros(1, device="cuda")
from webdnn_amd import capi, hostops as H
ctx = H.HipContext(0).initialize()
x = np.arange(12, dtype=np.float32).reshape(3, 4)
t, q = ctx.move_tensor(x), ctx.move_tensor(np.arange(5, dtype=np.uint8))
ctx.sync()
assert np.array_equal(torch.as_tensor(t, device="cuda").cpu().numpy(), x)
view = torch.as_tensor(q, device="cuda")
view += 1
torch.cuda.synchronize()
assert np.array_equal(q.get_data(), np.arange(1, 6))
assert torch.as_tensor(ctx.empty_tensor([0, 3]), device="cuda").shape == (0, 3)
for bad in ((t.handle, None), (12345678, capi.ctypes.byref(capi.ctypes.c_uint64()))):
    try:
        H.call("wdh_address", *bad)
        raise SystemExit("not refused")
    except capi.HipError as err:
        assert err.code == -2
print("same memory")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0 and "same memory" in done.stdout, done.stdout


# ---- together ------------------------------------------------------------------------------------
class Block:
    """One decoder block as a serving program runs it: everything between the residual stream's two ends in 8 bits."""

    def __init__(self, ctx, rng, width, heads, kv, d, hidden):
        self.ctx, self.heads, self.kv, self.d = ctx, heads, kv, d
        weight = lambda n, k: H.quantize_fp8(ctx, ctx.move_tensor((rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32)), 128)
        self.g1, self.g2 = (ctx.move_tensor(rng.uniform(0.5, 1.5, width).astype(np.float32)) for _ in range(2))
        self.qkv, self.o, self.up, self.down = weight((heads + 2 * kv) * d, width), weight(width, heads * d), weight(hidden, width), weight(width, hidden)

    def run(self, x, cache, table, lens, starts):
        ctx, hd = self.ctx, self.heads * self.d
        q8, c = H.rms_normalization_fp8(ctx, x, self.g1)
        qkv = H.matmul_fp8(ctx, q8, c, *self.qkv)
        H.cache_append(ctx, cache, qkv, qkv, table, lens, starts, k_column=hd, v_column=hd + self.kv * self.d)
        a = H.cache_attention(ctx, cache, qkv, self.heads, self.d ** -0.5, table, lens, starts)
        a8, ac = H.quantize_fp8(ctx, a)
        y = H.matmul_fp8(ctx, a8, ac, *self.o)
        s, n8, nc = H.rms_normalization_fp8(ctx, y, self.g2, x)
        u = H.matmul_fp8(ctx, n8, nc, *self.up, epilogue="relu")
        u8, uc = H.quantize_fp8(ctx, u)
        out = H.matmul_fp8(ctx, u8, uc, *self.down, residual=s)
        self.seen = dict(q8=q8, c=c, qkv=qkv, a=a, y=y, s=s, n8=n8, nc=nc, u=u, u8=u8, uc=uc, out=out)
        return out


def check_block(block, x, cache_before, cache, table, lens, starts):
    """Every step against its definition, on what the step before it left."""
    seen = {n: t.get_data() for n, t in block.seen.items()}
    n, hd, kd = x.shape[0], block.heads * block.d, block.kv * block.d
    F.check_quantized(seen["q8"], seen["c"], F.rms(x.astype(np.float64), block.g1.get_data().astype(np.float64), 1e-5), 1, 3.01 * E, "norm")

    def near(a, sa, w, want_for, extra=0.0):
        want, size = F.product(seen[a], seen[sa], *(t.get_data() for t in w))
        want = want + extra
        want = np.maximum(want, 0) if want_for == "u" else want
        bound = (128 + 4 + seen[sa].shape[1]) * 2 * E * size + E * np.abs(want)
        assert np.all(np.abs(seen[want_for] - want) <= bound), want_for

    near("q8", "c", block.qkv, "qkv")
    cache_before.append(seen["qkv"][:, hd:hd + kd].reshape(n, block.kv, block.d), seen["qkv"][:, hd + kd:].reshape(n, block.kv, block.d), table, lens, starts)
    check_cache(cache, cache_before)
    want, bound = cache_before.attention(seen["qkv"][:, :hd].reshape(n, block.heads, block.d), table, lens, starts, block.d ** -0.5)
    assert np.all(np.abs(seen["a"].reshape(want.shape) - want) <= bound)
    assert np.array_equal(seen["s"], seen["y"] + x)
    F.check_quantized(seen["n8"], seen["nc"], F.rms(seen["s"].astype(np.float64), block.g2.get_data().astype(np.float64), 1e-5), 1, 3.01 * E, "second norm")
    near("n8", "nc", block.up, "u")
    F.check_quantized(seen["u8"], seen["uc"], seen["u"].astype(np.float64), 1, 0.0, "u")
    near("u8", "uc", block.down, "out", seen["s"].astype(np.float64))


def test_a_block_serves_prompts_and_then_tokens(ctx):
    rng = np.random.default_rng(21)
    heads, kv, d, width, hidden = 6, 2, 64, 320, 1000
    block = Block(ctx, rng, width, heads, kv, d, hidden)
    table, _, _, pages = layout(rng, [90, 5, 70], [40, 60, 2])
    c = F.Cache(pages, kv, d)
    cache = on_device(ctx, c)
    lens = np.zeros(3, np.int32)
    for new in ([80, 3, 64], [1, 1, 1], [1, 1, 1], [20, 0, 2]):
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        lens = (lens + new).astype(np.int32)
        x = rng.standard_normal((int(starts[-1]), width)).astype(np.float32)
        block.run(ctx.move_tensor(x), cache, *(ctx.move_tensor(t) for t in (table, lens, starts)))
        check_block(block, x, c, cache, table, lens, starts)


def test_a_recorded_block_follows_its_sequences(ctx):
    """Recorded once, replayed with other tokens, lengths and tables in the same buffers; every replay against the node-by-node run."""
    rng = np.random.default_rng(22)
    heads, kv, d, width, hidden, seqs = 8, 2, 128, 256, 512, 3
    block = Block(ctx, rng, width, heads, kv, d, hidden)
    table, lens, _, pages = layout(rng, [8] * seqs, [150, 62, 900])
    lens, starts = (lens - 7).astype(np.int32), np.arange(4, dtype=np.int32)
    cache = H.KvCache.empty(ctx, pages, kv, d)
    twin = H.KvCache.empty(ctx, pages, kv, d)
    first = np.concatenate([[0], np.cumsum(lens - 1)]).astype(np.int32)
    k = ctx.move_tensor(rng.standard_normal((int(first[-1]), kv * d)).astype(np.float32))
    dt, dl, ds = ctx.move_tensor(table), ctx.move_tensor(lens), ctx.move_tensor(starts)
    for one in (cache, twin):
        H.cache_append(ctx, one, k, k, dt, ctx.move_tensor((lens - 1).astype(np.int32)), ctx.move_tensor(first))
    x = ctx.move_tensor(rng.standard_normal((seqs, width)).astype(np.float32))
    block.run(x, twin, dt, dl, ds)                                    # (the first run fills the pool)
    H.cache_append(ctx, twin, k, k, dt, ctx.move_tensor((lens - 1).astype(np.int32)), ctx.move_tensor(first))
    ctx.sync()
    ctx.graph_begin()
    out = block.run(x, cache, dt, dl, ds)
    graph = ctx.graph_end()
    try:
        for turn in range(4):
            rows = rng.standard_normal((seqs, width)).astype(np.float32)
            x.set_data(rows)
            dl.set_data(lens)
            ctx.graph_launch(graph)
            got = out.get_data()
            want = block.run(x, twin, dt, dl, ds)
            assert np.array_equal(got, want.get_data()), turn
            for a, b in ((cache.k_scales, twin.k_scales), (cache.v_scales, twin.v_scales)):
                assert np.array_equal(a.get_data()[table[0, :2]], b.get_data()[table[0, :2]])
            want.dispose()
            lens = (lens + 1).astype(np.int32)
            if turn == 1:                                             # sequences may change places
                table = table[::-1].copy()
                lens = lens[::-1].copy()
                dt.set_data(table)
    finally:
        ctx.graph_destroy(graph)
