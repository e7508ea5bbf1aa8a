"""The MXFP4 oracle against closed forms (CPU only)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import mxfp4 as omx


def test_levels_are_their_own_codes():
    t = np.concatenate([omx.LEVELS, -omx.LEVELS, np.full(16, 6.0)])[None]
    code, scales = omx.encode(t)
    assert scales.tolist() == [[127]]
    assert code[0, :16].tolist() == list(range(8)) + [8 | c for c in range(8)]
    assert np.array_equal(omx.values(t), t)


@pytest.mark.parametrize("value,code", [(0.25, 0), (0.2500001, 1), (0.75, 2), (1.25, 2), (1.75, 4),
                                        (2.5, 4), (3.5, 6), (5.0, 6), (5.0000001, 7), (7.99, 7)])
def test_ties_go_to_the_even_code_and_the_top_saturates(value, code):
    assert omx.nearest_code(np.array([value]))[0] == code


def test_scales_of_powers_zeros_and_extremes():
    t = np.zeros((8, 32))
    t[1, 3], t[2, 0], t[3, 31], t[4, 5] = 1.0, 8.0, 2.0 ** -126, 2.0 ** -149
    t[5, 1], t[6, 2], t[7, 9] = np.inf, np.nan, 3.3e38
    assert omx.scale_bytes(t)[:, 0].tolist() == [0, 125, 128, 0, 0, 255, 255, 252]
    v = omx.values(t)
    assert v[1, 3] == 1.0 and v[2, 0] == 8.0 and np.isnan(v[5]).all() and np.isnan(v[6]).all()
    assert v[3, 31] == 2.0 ** -126 and v[4, 5] == 0.0


def test_stored_layout():
    t = np.zeros((33, 300))
    t[32, 0], t[32, 1], t[32, 299] = 1.0, -1.5, 4.0
    codes, scales = omx.stored(t)
    assert codes.shape == (33, 256) and scales.shape == (2, 64, 8)
    # 1.0 = 4 * 2^-2 and -1.5 = -6 * 2^-2: low and high half of the first byte
    assert codes[32, 0] == (6 | (15 << 4)) and scales[0, 32, 0] == 125
    assert codes[32, 149] == 6 << 4 and scales[1, 32, 1] == 127
    assert scales[:, 33:].max() == 0


def test_gated_gradients_against_differences():
    g, u, dh = np.random.Generator(np.random.PCG64(3)).standard_normal((3, 5, 7)) * 3
    h = 1e-6
    dg, du = omx.gated_gradients(dh, g, u)
    np.testing.assert_allclose(dg, dh * (omx.gated(g + h, u) - omx.gated(g - h, u)) / (2 * h),
                               rtol=1e-7, atol=1e-8)
    np.testing.assert_allclose(du, dh * (omx.gated(g, u + h) - omx.gated(g, u - h)) / (2 * h),
                               rtol=1e-7, atol=1e-8)
