"""The 8-bit serving operators at operands where a definition and a shortcut part: quotients beside a tie, pages of
values that differ in size, scales that are no numbers."""
import numpy as np
import pytest
import torch

import fp8_ref as F
import test_gpu_fp8_serving as S
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu


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
