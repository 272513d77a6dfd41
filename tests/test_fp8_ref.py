"""The 64-bit restatement of the 8-bit operators (tests/fp8_ref.py) against torch's own e4m3 type and against differences."""
import numpy as np
import torch

import fp8_ref as F


def test_decode_is_torchs_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(F.VALUES)) and np.array_equal(t[~np.isnan(t)], F.VALUES[~np.isnan(t)])


def test_encode_is_the_nearest_value_and_ties_go_to_even():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(4000) * 2.0 ** rng.integers(-14, 9, 4000), VALUES_AND_MIDDLES(), [0.0, -0.0, 447.9, -460.0]])
    x = x[np.abs(x) <= 448].astype(np.float32).astype(np.float64)
    got = F.encode(x)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(got, want)
    assert np.array_equal(F.encode([np.inf, -np.inf, np.nan]) & 127, [127, 127, 127])


def VALUES_AND_MIDDLES():
    v = F.VALUES[:127]
    both = np.concatenate([v, (v[1:] + v[:-1]) / 2])
    return np.concatenate([both, -both])


def test_page_scales_are_the_least_powers_that_fit():
    amax = np.array([448.0, 448.0001, 1.0, 0.875, 0.8750001, 1e-37, 0.0, 3e38], np.float32)
    c = F.page_scale(amax)
    assert np.all(amax.astype(np.float64) <= 448 * c) and np.all((c == F.LEAST) | (amax.astype(np.float64) > 448 * c / 2))
    assert np.array_equal(np.log2(c), np.round(np.log2(c)))
