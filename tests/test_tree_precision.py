"""What the precision test of attention of trees is worth, without a GPU: its cases reach every form of items, and its bound rejects what a kernel
without the second parts of its queries or its weights would give."""
import numpy as np
import pytest

import fp8_ref as F
import tree_plan


@pytest.mark.parametrize("d", [32, 64, 128])
def test_the_cases_reach_every_form(d):
    forms = [tree_plan.form_of(*case, d) for case in tree_plan.CASES]
    assert sorted(forms) == [(rows, shared) for rows in (32, 64, 128) for shared in (False, True)]


def parts(x, n):
    """The sum of n float16 numbers, each the nearest to what the ones before leave."""
    held = np.zeros(x.shape)
    for _ in range(n):
        held = held + (x - held).astype(np.float16)
    return held


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("new,past,heads,kv", tree_plan.CASES)
def test_a_part_left_out_shows_in_the_2_norm(new, past, heads, kv, d):
    """Rows of one head of the cache, as the case's first sequence has them; queries are brought to 2^14 and weights to 2^8 before they are cut."""
    rng = np.random.default_rng(sum(new) + d)
    rows, keys = new[0] * heads // kv, new[0] + past[0]
    pool = F.decode(F.encode(rng.standard_normal(4099) * 64)) / 64
    k, v = (rng.choice(pool, (keys, d)) for _ in range(2))
    q = rng.standard_normal((rows, d)).astype(np.float32) * d ** -0.5
    up = 2.0 ** (14 - np.floor(np.log2(np.abs(q).max(1, keepdims=True))))

    def attention(of_q, of_w):
        t = (parts(q * up, of_q) if of_q else q * up) @ k.T / up
        w = 2.0 ** 8 * np.exp(t - t.max(1, keepdims=True))
        return (parts(w, of_w) if of_w else w) @ v / w.sum(1, keepdims=True)

    want = attention(0, 0)
    error = lambda *p: np.linalg.norm(attention(*p) - want) / np.linalg.norm(want)
    assert error(2, 2) < 2.0 ** -21
    assert error(1, 2) > 2.0 ** -20 and error(2, 1) > 2.0 ** -20
