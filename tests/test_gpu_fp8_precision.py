"""The precision that the 8-bit operators are built for: products in every form with sums that fp32 holds exactly, and in 2-norm; attention in
2-norm in every form."""
import numpy as np
import pytest

import fp8_plan
import fp8_ref as F
import test_gpu_fp8_edges as X
import test_gpu_fp8_serving as S
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", fp8_plan.CASES)
def test_every_form_of_the_products(ctx, m, n, k):
    """Against the worst case (with everything that is fused), and in 2-norm: the factor of a block's sum and its product are two roundings,
    the sums of K / 128 blocks that many more, independent of each other."""
    rng = np.random.default_rng(m + n + k)
    S.check_product(ctx, rng, m, n, k, bias=True, residual=m % 2 == 0, relu=n % 3 == 0)
    kb = -(-k // 128)
    a, w = F.encode(rng.standard_normal((m, k)) * 100), F.encode(rng.standard_normal((n, k)) * 100)
    sa, sw = (rng.uniform(0.5, 1, s).astype(np.float32) for s in ((m, kb), (-(-n // 128), kb)))
    want, _ = F.product(a, sa, w, sw)
    got = H.matmul_fp8(ctx, *(ctx.move_tensor(t) for t in (a, sa, w, sw))).get_data()
    assert X.relative(got, want) <= (2 + kb ** 0.5) * 2.0 ** -24, X.relative(got, want) * 2.0 ** 24


@pytest.mark.parametrize("m,n,k", fp8_plan.CASES)
def test_sums_of_whole_numbers_are_exact(ctx, m, n, k):
    """Products of 65536 beside products of 1: whole numbers below 2^24 in any order of addition, which fp32 sums hold."""
    rng = np.random.default_rng(m + n + k)
    kb = -(-k // 128)
    assert kb * (65536 + 127) < 2 ** 24
    large = np.zeros(k, bool)
    large[np.minimum(np.arange(kb) * 128 + rng.integers(0, 128, kb), k - 1)] = True
    signs = lambda *s: np.where(rng.random(s) < 0.5, -1.0, 1.0)
    a, w = (np.where(large, 256.0, 1.0) * signs(rows, k) for rows in (m, n))
    sa, sw = np.ones((m, kb), np.float32), np.ones((-(-n // 128), kb), np.float32)
    got = H.matmul_fp8(ctx, *(ctx.move_tensor(t) for t in (F.encode(a), sa, F.encode(w), sw))).get_data()
    assert np.array_equal(got, a @ w.T)


# single tokens in shares of pages, a workgroup to an item, one long sequence; parts of prompts in 16-row items; 128-row items whole and in parts
@pytest.mark.parametrize("new,past,heads,kv,d", [(1, 3000, 16, 2, 128), (1, 20000, 8, 1, 64), (3, 700, 8, 8, 32), (40, 300, 8, 2, 128), (200, 1000, 8, 4, 64),
                                                 (300, 0, 4, 1, 32), (700, 100, 32, 8, 128), (1300, 700, 64, 2, 32), (650, 30, 64, 64, 64), (330, 3000, 64, 1, 128)])
def test_attention(ctx, new, past, heads, kv, d):
    """(The bound: see test_values_of_pages_that_differ_in_size.)"""
    rng = np.random.default_rng(new + past)
    c, table, lens, starts = S.filled(rng, [new], [past], kv, d)
    q = rng.standard_normal((new, heads, d)).astype(np.float32)
    want = X.attention(c, q, table[0], int(lens[0]), d ** -0.5)
    got = S.attend(ctx, c, q, table, lens, starts, np.float32(d ** -0.5))
    assert X.relative(got, want) <= 2.0 ** -20, X.relative(got, want) * 2.0 ** 20


@pytest.mark.parametrize("m,n,k", [(71, 11770, 3792), (364, 70, 8176), (1384, 379, 3639), (5825, 147, 3798)])
def test_a_cut_product_without_room_for_its_parts(ctx, m, n, k):
    assert fp8_plan.plan(m, n, k)[1] > 1
    rng = np.random.default_rng(k)
    a, w = S.bytes_of(rng, (m, k)), S.bytes_of(rng, (n, k))
    kb = -(-k // 128)
    sa, sw = np.full((m, kb), 0.5, np.float32), np.full((-(-n // 128), kb), 0.25, np.float32)
    ops, y = [ctx.move_tensor(t) for t in (a, sa, w, sw)], ctx.empty_tensor([m, n])
    ctx.sync()
    H.call("wdh_trim", 0)
    ctx.set_option("memory_limit_mib", 1)
    try:
        H.matmul_fp8(ctx, *ops, out=y)
    finally:
        ctx.set_option("memory_limit_mib", 0)
    want, size = F.product(a, sa, w, sw)
    assert np.all(np.abs(y.get_data() - want) <= (128 + 2 + kb) * 2 * S.E * size)
