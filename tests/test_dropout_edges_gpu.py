"""Dropout's entry point at the ends of what its header allows (GPU)."""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd import _native as nat

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _launch(x, key, site, threshold, out):
    code = nat.DTYPE_BF16 if x.dtype == torch.bfloat16 else nat.DTYPE_F32
    args = (x.data_ptr(), code, x.numel(), None if key is None else key.data_ptr(), site, threshold,
            out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    nat.call("rpx_dropout", *args)
    nat.check(nat.fast().dropout(*args))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("count", [1, 7, 4099])
def test_no_dropout_needs_no_key(dtype, count):
    x = torch.randn(count, device=DEV).to(dtype)
    for key in (None, torch.tensor([3, 4], device=DEV)):
        out = torch.full_like(x, 7)
        _launch(x, key, 0, 65536, out)
        assert torch.equal(out, x)


def test_the_output_may_be_the_input():
    x = torch.randn(4099, device=DEV)
    key = torch.tensor([3, 4], device=DEV)
    want = rx.dropout(x, 0.5, key, 2)
    again = rx.dropout(want, 0.5, key, 2)  # the launch runs once for either binding
    _launch(x, key, 2, 32768, x)
    assert torch.equal(x, again)


@pytest.mark.parametrize("rate,threshold", [(1 - 2.0 ** -16, 1), (2.0 ** -16, 65535)])
def test_the_smallest_and_largest_thresholds(rate, threshold):
    key = torch.tensor([3, 4], device=DEV)
    x = torch.ones(1 << 20, device=DEV)
    y = rx.dropout(x, rate, key)
    kept = y != 0
    assert (y[kept] == 65536 / threshold).all()
    # binomial: six deviations
    p, n = threshold / 65536, x.numel()
    assert abs(int(kept.sum()) - n * p) <= 6 * (n * p * (1 - p)) ** 0.5
