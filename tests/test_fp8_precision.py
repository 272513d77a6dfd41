"""What the precision tests of the 8-bit operators are worth, without a GPU: their product cases reach every form there is, and their bounds
reject what a kernel with a part of its operands left out, or on the 8-bit matrix instructions, would give."""
import math
import random

import numpy as np

import fp8_plan
import fp8_ref as F


def test_the_cases_reach_every_form_that_sizes_can():
    rng = random.Random(1)
    reached = set()
    for _ in range(60000):
        m, n, k = (int(round(math.exp(rng.uniform(0, math.log(most))))) for most in (20000, 20000, 30000))
        reached.add(fp8_plan.kind(m, n, max(16, k // 16 * 16) if rng.random() < 0.5 else k))
    covered = [fp8_plan.kind(*case) for case in fp8_plan.CASES]
    assert set(covered) >= reached, sorted(map(str, reached - set(covered)))
    assert len(set(covered)) == len(covered) == 4 * len(fp8_plan.FORMS) + 4


def _cut(x, bits, parts):
    """fp32 numbers as `parts` terms of `bits` significant bits each, rounded towards zero."""
    left, out = x.astype(np.float64), 0.0
    for _ in range(parts):
        e = np.floor(np.log2(np.maximum(np.abs(left), 2.0 ** -200)))
        part = np.trunc(left / 2.0 ** (e - bits + 1)) * 2.0 ** (e - bits + 1)
        out, left = out + part, left - part
    return out


def _attention(q, k, v, weights=lambda p: p):
    t = q @ k.T * 0.125
    p = np.exp(t - t.max(1, keepdims=True))
    return weights(p) @ v / p.sum(1, keepdims=True)


def test_a_part_of_queries_or_weights_left_out_shows_in_the_2_norm():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((n, 64)).astype(np.float32) for n in (40, 1500, 1500))
    k, v = F.decode(F.encode(k * 64)) / 64, F.decode(F.encode(v * 64)) / 64
    want = _attention(q.astype(np.float64), k, v)
    error = lambda got: np.linalg.norm(got - want) / np.linalg.norm(want)
    for bits, parts in ((8, 3), (11, 2)):                                    # bfloat16 in three, float16 in two
        whole, less = (lambda x, n=n: _cut(x, bits, n) for n in (parts, parts - 1))
        assert error(_attention(whole(q), k, v, whole)) < 2.0 ** -21
        assert error(_attention(less(q), k, v)) > 2.0 ** -20
        assert error(_attention(q.astype(np.float64), k, v, less)) > 2.0 ** -20


def _eight_bit_block(a, w):
    """A block's sums as the 8-bit matrix instructions give them: of each group of eight products what lies 15 bits and more below the
    largest is left out."""
    products = (a[:, None, :] * w[None, :, :]).reshape(len(a), len(w), -1, 8)
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(products).max(-1, keepdims=True), 2.0 ** -60))) - 15)
    return (np.trunc(products / step) * step).sum((-1, -2))


def test_the_8_bit_instructions_would_show():
    row = np.ones((1, 128))
    big = row.copy()
    big[0, 5] = 256
    assert _eight_bit_block(big, big)[0, 0] == 65656                         # (as they do on the device; 65663 it is)
    rng = np.random.default_rng(1)
    a, w = (F.decode(F.encode(rng.standard_normal((30, 128)) * 100)) for _ in range(2))
    want = a @ w.T
    assert np.linalg.norm(_eight_bit_block(a, w) - want) / np.linalg.norm(want) > 3 * 2.0 ** -24
