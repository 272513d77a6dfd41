"""The operators for drafted tokens at operands where a definition and a shortcut part: zeros kept from pages of large scales."""
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
