"""The generator against its published vectors, dropout by torch operations
against the oracle, and refusals (CPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import representax_amd as rx
from oracle import dropout as odrop
from representax_amd import _native as nat
from representax_amd.philox import dropout_threshold, dropped, kept


# counter, key and result of the generator's authors' known answers
@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_philox_known_answers(counter, key, want):
    got = odrop.philox4x32([np.uint64(c) for c in counter], key)
    assert tuple(int(w) for w in got) == want


@pytest.mark.parametrize("count", [1, 7, 8, 9, 1003])
@pytest.mark.parametrize("seed,step,site", [(0, 0, 0), (1 << 62, 3, 7),
                                            (0x123456789ABCDEF, 2 ** 32 - 1, 2 ** 32 - 1)])
def test_expression_equals_oracle(count, seed, step, site):
    key = torch.tensor([seed, step])
    for below in (1, 30000, 65535):
        want = odrop.kept(count, seed, step, site, below)
        got = kept((count,), key, below, site).numpy()
        assert np.array_equal(got, want)


def test_rate_is_kept_and_expectation_is_exact():
    key = rx.DropoutKeys(11).next()
    x = torch.ones(1 << 18, dtype=torch.float64)
    for rate in (0.1, 0.5, 0.9):
        y = rx.dropout(x, rate, key)
        p = 1 - dropout_threshold(rate) / 65536
        # mean of 2^18 independent values of variance p / (1 - p): six deviations
        assert abs(y.mean().item() - 1) < 6 * (p / (1 - p) / x.numel()) ** 0.5
        assert set(y.unique().tolist()) == {0.0, 1 / (1 - p)}


def test_keys_sites_and_steps_differ():
    keys = rx.DropoutKeys(5)
    a, b = keys.next(), keys.next()
    x = torch.ones(4096)
    masks = [rx.dropout(x, 0.5, k, site) for k in (a, b) for site in (0, 1)]
    for i in range(4):
        for j in range(i):
            # independent halves agree on 2048 of 4096, deviation 32
            agree = (masks[i] == masks[j]).sum().item()
            assert abs(agree - 2048) < 6 * 32
    assert torch.equal(rx.dropout(x, 0.5, a, 1), masks[1])
    assert a.tolist() == [5, 1] and b.tolist() == [5, 2]


def test_gradient_is_the_same_mask_and_composes():
    key = rx.DropoutKeys(3).next()
    x = torch.randn(5, 13, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: rx.dropout(t, 0.3, key, 2), (x,))
    assert torch.autograd.gradgradcheck(lambda t: rx.dropout(t, 0.3, key, 2) ** 2, (x,))
    assert rx.dropout(x, 0.0, None) is x


def test_dropped_values_are_zero_whatever_they_were():
    key = torch.tensor([1, 1])
    x = torch.tensor([float("nan"), float("inf")] * 32)
    keep = kept(x.shape, key, 32768, 0)
    y = dropped(x, key, 32768, 0)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


@pytest.mark.parametrize("rate", [-0.1, 1.0, 1.5, float("nan")])
def test_rates_outside_are_refused(rate):
    with pytest.raises(ValueError, match="rate"):
        rx.dropout(torch.ones(4), rate, torch.zeros(2, dtype=torch.int64))


def test_bad_keys_and_values_are_refused():
    x = torch.ones(4)
    with pytest.raises(ValueError, match="key"):
        rx.dropout(x, 0.5, None)
    with pytest.raises(ValueError, match="key"):
        rx.dropout(x, 0.5, torch.zeros(2))
    with pytest.raises(ValueError, match="key"):
        rx.dropout(x, 0.5, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="site"):
        rx.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64), site=-1)
    with pytest.raises(TypeError):
        rx.dropout(torch.ones(4, dtype=torch.int32), 0.5, torch.zeros(2, dtype=torch.int64))


def test_entry_point_refuses_before_any_launch():
    p = ctypes.c_void_p(16)
    bf16 = nat.DTYPE_BF16
    for args, match in [((p, 9, 8, p, 0, 5, p), "dtype"), ((p, bf16, -1, p, 0, 5, p), "count"),
                        ((p, bf16, 8, p, 0, 0, p), "threshold"),
                        ((p, bf16, 8, p, 0, 65537, p), "threshold"),
                        ((p, bf16, 8, p, 1 << 32, 5, p), "site"),
                        ((p, bf16, 8, None, 0, 5, p), "key"),
                        ((p, bf16, 8, ctypes.c_void_p(12), 0, 5, p), "key"),
                        ((None, bf16, 8, p, 0, 5, p), "null"),
                        ((ctypes.c_void_p(18), bf16, 8, p, 0, 5, p), "aligned")]:
        with pytest.raises(ValueError, match=match):
            nat.call("rpx_dropout", *args, None)
    nat.call("rpx_dropout", None, bf16, 0, p, 0, 5, None, None)  # nothing to do
