"""The 8-bit serving operators where their forms change and where they end: every tile of the products, many sequences, caches
beyond 4 GiB, scales that are none, sequences that contradict each other, no room for a workspace, several recorded runs."""
import numpy as np
import pytest

import fp8_ref as F
import test_gpu_fp8_serving as S
from webdnn_amd import capi
from webdnn_amd import hostops as H

pytestmark = pytest.mark.gpu


# few rows by 16, 32 and 64 columns; 64 x 64; 128 x 128 with rows that are copied first, and more of them than the chip takes at
# once; 256 x 128; and cut along K, the last part being shorter, with and without whole 16-byte rows
@pytest.mark.parametrize("m,n,k", [(20, 1000, 12000), (100, 900, 9001), (300, 700, 14336), (500, 2000, 5000), (260, 1024, 16384), (2, 130, 20001), (16, 5000, 272), (3, 20000, 260), (11, 9000, 1030), (600, 1500, 400), (1500, 2000, 130), (3000, 2900, 144), (8192, 4096, 200)])
def test_every_tile_of_the_products(ctx, m, n, k):
    S.check_product(ctx, np.random.default_rng(m + n + k), m, n, k, bias=True, residual=m < 2000)


@pytest.mark.parametrize("n,k", [(1, 1), (3, 15), (130, 1023), (9001, 4100), (300, 14336), (257, 5000), (128, 1024), (5, 4097)])
def test_products_of_one_row(ctx, n, k):
    rng = np.random.default_rng(n + k)
    S.check_product(ctx, rng, 1, n, k, bias=True, residual=True, relu=True)
    a, w = S.bytes_of(rng, (1, k)), S.bytes_of(rng, (n, k))
    sa, sw = np.ones((1, -(-k // 128)), np.float32), np.ones((-(-n // 128), -(-k // 128)), np.float32)
    w[n // 2, k - 1] = 0xff
    up = ctx.move_tensor
    y = H.matmul_fp8(ctx, up(a), up(sa), up(w), up(sw)).get_data()
    assert np.array_equal(np.isnan(y[0]), np.arange(n) == n // 2)


@pytest.mark.parametrize("rows,length", [(9, 700), (6, 768), (1030, 769), (11, 1400), (3, 1536), (70, 1537), (2, 5000), (3, 6144), (40, 6145), (600, 8500), (5, 12000),
                                         (2, 16384), (513, 9001), (3, 16385)])
def test_every_form_of_the_norm(ctx, rows, length):
    S.test_norm(ctx, rows, length, True, True)


@pytest.mark.parametrize("cols", [3, 5, 20, 33, 64, 65, 100, 132, 137, 156, 190, 193])
def test_narrow_last_blocks(ctx, cols):
    rng = np.random.default_rng(cols)
    x = (rng.standard_normal((1300, cols)) * 2.0 ** rng.integers(-20, 20, (1300, 1))).astype(np.float32)
    q, c = (t.get_data() for t in H.quantize_fp8(ctx, ctx.move_tensor(x), 128))
    F.check_quantized(q, c, x.astype(np.float64), 128, 0.0)


@pytest.mark.parametrize("new,heads,kv,d", [([1, 0, 2] * 45, 4, 2, 32), ([20] * 70, 8, 2, 64), ([1] * 200, 3, 3, 64)])
@pytest.mark.parametrize("longest", [350, 900, 1500])          # (a workgroup to an item; the same for many items; shares of all pages)
def test_attention_of_more_sequences_than_lanes(ctx, new, heads, kv, d, longest):
    rng = np.random.default_rng(len(new))
    past = rng.integers(0, 350, len(new))
    past[5], past[66] = longest, 0
    c, table, lens, starts = S.filled(rng, new, past, kv, d)
    q = rng.standard_normal((int(starts[-1]), heads, d)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, d ** -0.5)
    assert np.all(np.abs(S.attend(ctx, c, q, table, lens, starts, np.float32(d ** -0.5)) - want) <= bound)


# Items of 128 rows (calls of 80 * 256 rows of queries of 128 elements and more): one long sequence cut into parts, several with short and
# empty ones between them, a head of the cache for each query, one for 64, more sequences than lanes
MANY = [([1300], [700], 64, 2, 32), ([600, 251, 1, 0, 40], [0, 65, 500, 0, 0], 48, 3, 64), ([1300], [0], 16, 4, 128), ([700, 600], [30, 1], 64, 64, 32),
        ([330], [3000], 64, 1, 128), ([20] * 70, list(range(0, 210, 3)), 30, 2, 64), ([900, 300, 50], [10, 0, 700], 24, 8, 128)]


@pytest.mark.parametrize("new,past,heads,kv,d", MANY)
def test_attention_of_many_rows(ctx, new, past, heads, kv, d):
    assert sum(new) * heads * d >= 80 * 128 * 256 and sum(new) * heads // kv >= 64 * len(new)
    rng = np.random.default_rng(sum(new))
    c, table, lens, starts = S.filled(rng, new, past, kv, d)
    q = rng.standard_normal((int(starts[-1]), heads, d)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, d ** -0.5)
    got = S.attend(ctx, c, q, table, lens, starts, np.float32(d ** -0.5), wide=4 * (len(new) % 2))
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))


def test_many_rows_with_sharp_scores(ctx):
    rng = np.random.default_rng(8)
    c, table, lens, starts = S.filled(rng, [650, 2], [40, 400], 2, 64)
    q = rng.standard_normal((652, 64, 64)).astype(np.float32) * np.float32(50)
    q[3] = 0
    want, bound = c.attention(q, table, lens, starts, -1.0)
    assert np.all(np.abs(S.attend(ctx, c, q, table, lens, starts, -1.0) - want) <= bound)


@pytest.mark.parametrize("new", [90, 650])
@pytest.mark.parametrize("size", [2.0 ** -70, 2.0 ** -95, 2.0 ** 100])
def test_tiny_and_huge_keys_and_queries(ctx, new, size):
    """Scores that are nothing next to each other, queries of zeros, and a page that only the last rows see and that is not there."""
    rng = np.random.default_rng(24)
    kv, d, heads = 2, 64, 64
    table, lens, starts, pages = S.layout(rng, [new], [30])
    c = F.Cache(pages, kv, d)
    k, v = (rng.standard_normal((int(lens[0]), kv, d)).astype(np.float32) for _ in range(2))
    c.append(k * np.float32(size), v, table, lens, [0, int(lens[0])])
    q = (rng.standard_normal((new, heads, d)) * min(1.0, 2.0 ** 20 / size)).astype(np.float32)
    q[5] = 0
    q[6:9] *= np.float32(2.0 ** -60)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    last = (int(lens[0]) - 1) // 64
    table[0, last] = -1
    got = S.attend(ctx, c, q, table, lens, starts, 0.125)
    seen = 64 * last - 30
    assert np.all(np.abs(got - want)[:seen] <= bound[:seen]) and np.isnan(got[seen:]).all()


def test_nan_behind_a_row_of_many_does_not_reach_it(ctx):
    rng = np.random.default_rng(9)
    c, table, lens, starts = S.filled(rng, [650], [30], 2, 64)
    q = rng.standard_normal((650, 64, 64)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    for hit, where in ((110, 5), (667, 40)):                             # a page in the middle and the last one
        page, slot = table[0, hit // 64], hit % 64
        c.v[page, 0, where, slot] = 0x7f
        c.k[page, 1, slot, 9] = 0xff
    got = S.attend(ctx, c, q, table, lens, starts, 0.125)
    rows = np.arange(650)[:, None, None] + 30
    nan = np.zeros(got.shape, bool)
    nan[:, :32, 5], nan[:, :32, 40], nan[:, 32:] = rows[..., 0] >= 110, rows[..., 0] >= 667, rows >= 110
    assert np.isnan(got[nan]).all() and np.all((np.abs(got - want) <= bound)[~nan])


@pytest.mark.parametrize("scale", [0.0, -1.0, np.inf, np.nan])
@pytest.mark.parametrize("values", [False, True])
def test_many_rows_and_a_page_without_a_scale_or_a_place(ctx, scale, values):
    rng = np.random.default_rng(14)
    c, table, lens, starts = S.filled(rng, [650, 1], [100, 70], 2, 64)
    q = rng.standard_normal((651, 64, 64)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    (c.vs if values else c.ks)[table[0, 3], 1] = scale                    # tokens 192 .. 255 of one head
    table[0, 6] = -5                                                      # tokens 384 .. 447 of both
    got = S.attend(ctx, c, q, table, lens, starts, 0.125)
    rows = np.arange(651)[:, None, None] + 100
    nan = np.broadcast_to((rows >= 384) & (rows < 750), got.shape).copy()
    nan[:, 32:] |= ((rows >= 192) & (rows < 750))
    assert np.isnan(got[nan]).all() and np.all((np.abs(got - want) <= bound)[~nan])


def test_a_cache_beyond_4_gib(ctx):
    """Keys alone take 4.3 GiB: pages on both sides of 2 and 4 GiB, tokens one by one and in a prompt."""
    rng = np.random.default_rng(31)
    heads, kv, d, pages = 16, 8, 128, 70000
    far = np.full((3, 18), -1, np.int32)
    far[0, :3], far[1, 0], far[2] = [69999, 32768, 65535], 65536, np.append([32767, 1], 66000 + np.arange(16))
    near = np.where(far < 0, -1, np.cumsum(far >= 0).reshape(far.shape) - 1).astype(np.int32)
    lens, starts = np.array([150, 1, 1140], np.int32), np.array([0, 150, 151, 1291], np.int32)
    k, v = (rng.standard_normal((1291, kv, d)).astype(np.float32) for _ in range(2))
    c = F.Cache(22, kv, d)
    c.append(k, v, near, lens, starts)
    cache = H.KvCache.empty(ctx, pages, kv, d)
    up = ctx.move_tensor
    H.cache_append(ctx, cache, up(k.reshape(1291, -1)), up(v.reshape(1291, -1)), up(far), up(lens), up(starts))
    for scales, want in ((cache.k_scales, c.ks), (cache.v_scales, c.vs)):
        assert np.array_equal(scales.get_data()[far[far >= 0]], want[near[near >= 0]])
    for begin in (starts, np.array([0, 1, 2, 3], np.int32)):                    # the prompts; their last tokens alone
        q = rng.standard_normal((int(begin[-1]), heads, d)).astype(np.float32)
        want, bound = c.attention(q, near, lens, begin, 0.1)
        got = H.cache_attention(ctx, cache, up(q.reshape(len(q), -1)), heads, 0.1, up(far), up(lens), up(begin)).get_data().reshape(q.shape)
        assert np.all(np.abs(got - want) <= bound)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        t.dispose()
    ctx.sync()
    capi.call("wdh_trim", 0)


@pytest.mark.parametrize("scale", [0.0, -1.0, np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("values", [False, True])
def test_a_scale_that_is_none_makes_its_rows_nan(ctx, scale, new, values):
    rng = np.random.default_rng(14)
    c, table, lens, starts = S.filled(rng, [new], [100], 2, 64)
    q = rng.standard_normal((new, 4, 64)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    (c.vs if values else c.ks)[table[0, 1], 1] = scale                          # tokens 64 .. 127 of one head: rows from 64 on see them
    got = S.attend(ctx, c, q, table, lens, starts, 0.125)
    assert np.all(np.abs(got - want)[:, :2] <= bound[:, :2]) and np.isnan(got[:, 2:]).all()


def test_sequences_that_contradict_each_other(ctx):
    """Every other sequence claims all rows of the call: 2^31 units of work, which no call with sequences behind each other has.  Rows that
    more than one sequence claims may hold anything; the call ends, and the next one is right."""
    seqs, tokens, heads, pages = 1024, 60 * 1024, 1, 4096
    starts = np.zeros(seqs + 1, np.int32)
    starts[1::2] = tokens
    lens = np.full(seqs, 64 * pages, np.int32)
    up = ctx.move_tensor
    cache = H.KvCache.empty(ctx, 1, 1, 32)
    q = ctx.empty_tensor([tokens, 32])
    y = H.cache_attention(ctx, cache, q, heads, 1.0, up(np.full((seqs, pages), -1, np.int32)), up(lens), up(starts))
    ctx.sync()
    y.dispose()
    rng = np.random.default_rng(3)
    c, table, lens, starts = S.filled(rng, [1, 2], [300, 7], 1, 32)
    q = rng.standard_normal((3, 2, 32)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.2)
    assert np.all(np.abs(S.attend(ctx, c, q, table, lens, starts, 0.2) - want) <= bound)


def test_no_room_for_a_workspace(ctx):
    """Attention that needs one fails and leaves no trace; a product that would copy its operands goes without."""
    rng = np.random.default_rng(6)
    c, table, lens, starts = S.filled(rng, [1], [2000], 4, 128)
    q = rng.standard_normal((1, 8, 128)).astype(np.float32)
    want, bound = c.attention(q, table, lens, starts, 0.1)
    up = ctx.move_tensor
    cache, ints, rows = S.on_device(ctx, c), [up(t) for t in (table, lens, starts)], up(q.reshape(1, -1))
    y = ctx.empty_tensor([1, 1024])
    m, n, k = 1500, 2000, 130
    a, w = S.bytes_of(rng, (m, k)), S.bytes_of(rng, (n, k))
    sa, sw = np.full((m, 2), 0.5, np.float32), np.full((16, 2), 0.25, np.float32)
    ops, product = [up(t) for t in (a, sa, w, sw)], ctx.empty_tensor([m, n])
    ctx.sync()
    capi.call("wdh_trim", 0)
    ctx.set_option("memory_limit_mib", 1)
    try:
        with pytest.raises(capi.HipError) as err:
            H.cache_attention(ctx, cache, rows, 8, 0.1, *ints, out=y)
        assert err.value.code == -3
        H.matmul_fp8(ctx, *ops, out=product)
    finally:
        ctx.set_option("memory_limit_mib", 0)
    sums, size = F.product(a, sa, w, sw)
    assert np.all(np.abs(product.get_data() - sums) <= (128 + 2 + 2) * 2 * S.E * size)
    got = H.cache_attention(ctx, cache, rows, 8, 0.1, *ints, out=y).get_data().reshape(q.shape)
    assert np.all(np.abs(got - want) <= bound)


def test_recorded_runs_do_not_share_workspaces(ctx):
    """Recorded calls with workspaces (shares of single tokens, parts of prompts, copied operands), replayed in turn with eager
    work of the same kinds and other allocations between them: every replay against the first results."""
    rng = np.random.default_rng(17)
    up = ctx.move_tensor
    calls = []
    for new, past in (([1, 1], [3000, 40]), ([100], [900]), ([1000, 300], [60, 0])):
        c, table, lens, starts = S.filled(rng, new, past, 2, 64)
        operands = (S.on_device(ctx, c), up(rng.standard_normal((sum(new), 2048)).astype(np.float32)), up(table), up(lens), up(starts))
        calls.append(lambda o=operands, out=None: H.cache_attention(ctx, o[0], o[1], 32, 0.125, *o[2:], out=out))
    a, w = up(S.bytes_of(rng, (1500, 130))), up(S.bytes_of(rng, (2000, 130)))
    sa, sw = ctx.move_tensor(np.full((1500, 2), 0.5, np.float32)), up(np.full((16, 2), 0.25, np.float32))
    calls.append(lambda out=None: H.matmul_fp8(ctx, a, sa, w, sw, out=out))
    want = [call().get_data() for call in calls]
    graphs, outs = [], []
    try:
        for call in calls:
            ctx.graph_begin()
            outs.append(call())
            graphs.append(ctx.graph_end())
        for turn in range(3):
            noise = up(np.full(1 << 20, np.nan, np.float32))
            for g in graphs[::1 if turn % 2 else -1]:
                ctx.graph_launch(g)
            eager = [call() for call in calls]
            for out, again, first in zip(outs, eager, want):
                assert np.array_equal(out.get_data(), first) and np.array_equal(again.get_data(), first)
                again.dispose()
            assert np.isnan(noise.get_data()).all()
            noise.dispose()
    finally:
        for g in graphs:
            ctx.graph_destroy(g)


def test_a_side_lane_takes_recorded_attention_only(ctx):
    rng = np.random.default_rng(18)
    c, table, lens, starts = S.filled(rng, [1, 3], [900, 20], 2, 64)
    up = ctx.move_tensor
    cache, q, ints = S.on_device(ctx, c), up(rng.standard_normal((4, 256)).astype(np.float32)), [up(t) for t in (table, lens, starts)]
    run = lambda: H.cache_attention(ctx, cache, q, 4, 0.125, *ints)
    want = run().get_data()
    ctx.set_lane(1)
    try:
        with pytest.raises(capi.HipError) as err:
            run()
        assert "recorded work only" in str(err.value)
        ctx.graph_begin()
        out = run()
        graph = ctx.graph_end()
        for _ in range(3):
            ctx.graph_launch(graph)
            assert np.array_equal(out.get_data(), want)
    finally:
        ctx.set_lane(0)
    ctx.graph_launch(graph)
    assert np.array_equal(out.get_data(), want)
    ctx.graph_destroy(graph)


def test_what_is_too_large_or_empty_is_refused(ctx):
    f, i, e = lambda *s: ctx.empty_tensor(s), lambda *s: ctx.empty_tensor(s, "int32"), lambda *s: ctx.empty_tensor(s, "float8e4m3fn")
    cache = H.KvCache(ctx, e(0, 1, 64, 32), f(0, 1), e(0, 1, 32, 64), f(0, 1))
    with pytest.raises(capi.HipError) as err:                                  # rows that see no page of it
        H.cache_attention(ctx, cache, f(1, 32), 1, 1.0, i(1, 1), i(1), i(2))
    assert err.value.code == -2 and "without pages" in str(err.value)
    H.cache_append(ctx, cache, f(1, 32), f(1, 32), i(1, 1), i(1), i(2))        # nothing to write to
    for m, n, k in ((1, (1 << 28) + 1, 1), (1 << 31, 1, 1), (1, 1, (1 << 30) + 1)):
        with pytest.raises(capi.HipError) as err:
            H.call("wdh_gemm_fp8", 1, 1, 1, 1, 0, 1, m, n, k, 0, 0)
        assert err.value.code == -2 and "too many" in str(err.value)
