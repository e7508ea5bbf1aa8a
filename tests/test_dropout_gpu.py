"""Dropout on the GPU, bit for bit against the oracle's mask."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import representax_amd as rx
from oracle import dropout as odrop
from representax_amd import _native as nat
from tests.helpers import kernel_names

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _want(x, rate, key, site):
    seed, step = key.tolist()
    below = odrop.threshold(rate)
    keep = odrop.kept(x.numel(), seed, step, site, below)
    keep = torch.from_numpy(keep).to(x.device).view(x.shape)
    # one product in float32 and one rounding to the type
    return torch.where(keep, x.float() * np.float32(65536.0 / below), 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 683), (2049,), (5, 7, 64)])
@pytest.mark.parametrize("rate", [0.1, 0.75])
def test_values_and_gradient(dtype, shape, rate):
    g = torch.Generator().manual_seed(len(shape))
    x = torch.randn(shape, generator=g).to(DEV, dtype).requires_grad_(True)
    dy = torch.randn(shape, generator=g).to(DEV, dtype)
    key = rx.DropoutKeys(1234567890123, DEV).next()
    (y, (dx,)), names = kernel_names(
        lambda: (lambda y: (y, torch.autograd.grad(y, x, dy)))(rx.dropout(x, rate, key, 9)))
    assert sum("k_dropout" in n for n in names) >= 1
    assert torch.equal(y.detach(), _want(x.detach(), rate, key, 9))
    assert torch.equal(dx, _want(dy, rate, key, 9))


def test_views_empty_tensors_and_other_types():
    key = rx.DropoutKeys(4, DEV).next()
    base = torch.randn(33, 40, device=DEV)
    for x in (base.t(), base[:, 1:], base[1::2, ::3], base.view(-1)[1:], base.half(),
              base.double()):
        got = rx.dropout(x, 0.4, key)
        if x.dtype == torch.float64:
            keep = _want(torch.ones(x.shape, device=DEV), 0.4, key, 0) != 0
            assert torch.equal(got, torch.where(keep, x * (65536 / odrop.threshold(0.4)), 0.0))
        else:
            assert torch.equal(got, _want(x.contiguous(), 0.4, key, 0))
    assert rx.dropout(base[:0], 0.4, key).shape == (0, 40)


def test_elements_beyond_32_bit_counters():
    """The last elements of a tensor of more than 2^32 values."""

    count = (1 << 32) + 8 * 1024 + 5
    x = torch.ones(count, dtype=torch.bfloat16, device=DEV)
    key = torch.tensor([77, 3], device=DEV)
    y = rx.dropout(x, 0.5, key, 1)
    for first in (0, (1 << 32) - 16, (1 << 32) + 3, count - 1005):
        want = odrop.kept(1000, 77, 3, 1, 32768, first)
        assert np.array_equal((y[first:first + 1000] != 0).cpu().numpy(), want)


def test_second_derivative_and_frozen_input():
    key = rx.DropoutKeys(8, DEV).next()
    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    y = rx.dropout(x, 0.3, key)
    (dx,) = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    factor = _want(torch.ones_like(x.detach()), 0.3, key, 0)
    torch.testing.assert_close(ddx, 2 * factor ** 2)
    assert not rx.dropout(x.detach(), 0.3, key).requires_grad


def test_a_captured_step_draws_anew_each_replay():
    keys = rx.DropoutKeys(21, DEV)
    x = torch.randn(64, 256, device=DEV).to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn_like(x)

    def step():
        key = keys.next()
        y = rx.dropout(x, 0.2, key, 4)
        return key, y.detach(), *torch.autograd.grad(y, x, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        key, y, dx = step()
    seen = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.randn(1000, device=DEV).sum()  # the program's own work between replays
        assert torch.isfinite(eager)
        assert torch.equal(y, _want(x.detach(), 0.2, key, 4))
        assert torch.equal(dx, _want(dy, 0.2, key, 4))
        seen.append(key.tolist()[1])
    assert seen == list(range(seen[0], seen[0] + 4))


def test_an_unaligned_key_is_taken():
    keys = torch.tensor([0, 5, 6], device=DEV)
    x = torch.randn(100, device=DEV)
    assert torch.equal(rx.dropout(x, 0.5, keys[1:]), _want(x, 0.5, keys[1:], 0))
    assert nat.load() is not None
