"""Banks round y and dx once (GPU).

Small whole numbers, and quarters of them, whose sums float32 holds exactly in any
order: h and dh are bf16 values, so y and dx are the exact sums rounded once to bf16,
bit for bit. A base product rounded before the adapter's term, or before the bias,
ends elsewhere for many elements.
"""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd import ops

pytestmark = pytest.mark.gpu
DEV, BF16, F64 = "cuda:0", torch.bfloat16, torch.float64
ADAPTERS = 5


def _whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g).to(F64)


def _picks(g, rank, columns):
    """Rows [rank, columns] of one 1 each: a product with them picks values."""

    at = torch.randint(0, columns, (ADAPTERS, rank), generator=g)
    return torch.nn.functional.one_hot(at, columns).to(F64)


class Exact:
    def __init__(self, m, k, n, rank, group):
        g = torch.Generator().manual_seed(m + k + n + rank)
        q = torch.randint(-7, 8, (n, k), generator=g)
        nibbles = torch.nn.functional.pad(q & 15, (0, k % 2))
        self.packed = (nibbles[:, ::2] | (nibbles[:, 1::2] << 4)).to(torch.uint8).to(DEV)
        self.scales = torch.ones((n, k // group if group else 1), dtype=BF16).view(torch.int16).view(
            torch.uint16).to(DEV)
        self.w = q.to(F64)
        self.bias = _whole(g, 31, n) / 4
        # h = 2 x[c] (a kept element of a dropout of a half) is exact, y's term whole eighths
        self.x, self.dy = _whole(g, 7, m, k), _whole(g, 7, m, n)
        self.a, self.b = _picks(g, rank, k), _whole(g, 31, ADAPTERS, n, rank) / 4
        # and dh = g[c], dx's term the same
        self.at, self.bt = _whole(g, 31, ADAPTERS, rank, k) / 4, _picks(g, rank, n).transpose(1, 2)
        self.index = torch.randint(-1, ADAPTERS, (m,), generator=g)
        self.s = torch.tensor([0.5, 1.0, 0.25, 2.0, 0.5])
        self.group = group
        self.key = torch.tensor([5, 9], device=DEV)

    def call(self, x, a, b, rate):
        return rx.bank_linear(x, self.packed, self.scales, a.to(DEV, BF16), b.to(DEV, BF16),
                              self.s.to(DEV), rx.adapter_plan(self.index, ADAPTERS, DEV),
                              group_size=self.group, bias=self.bias.to(DEV, BF16), rate=rate,
                              key=self.key, site=3)

    def check(self, rate):
        x = self.x.to(DEV, BF16).requires_grad_(True)
        factor = torch.ones_like(self.x)
        if rate:
            factor = rx.dropout(torch.ones_like(self.x, device=DEV), rate, self.key, 3).cpu()
        e, on = self.index.clamp_min(0), (self.index >= 0).to(F64) * self.s.to(F64)[self.index]
        pick = lambda v, p: (v[:, None] * p[e]).sum(2)  # [m, rank] of [m, c] and [m, rank, c]
        h = pick(self.x * factor, self.a)
        y = self.x @ self.w.t() + self.bias + on[:, None] * (h[:, None] * self.b[e]).sum(2)
        assert y.abs().max() < 1 << 20 and torch.equal(y * 16, (y * 16).round())
        with torch.no_grad():
            got = [self.call(x, self.a, self.b, rate)]
        got.append(self.call(x, self.a, self.b, rate).detach())  # with h kept
        for v in got:
            assert torch.equal(v.cpu(), y.to(torch.float32).to(BF16))
        dh = pick(self.dy, self.bt.transpose(1, 2))
        dx = self.dy @ self.w + on[:, None] * (dh[..., None] * self.at[e]).sum(1) * factor
        assert dx.abs().max() < 1 << 20 and torch.equal(dx * 16, (dx * 16).round())
        (got,) = torch.autograd.grad(self.call(x, self.at, self.bt, rate), x,
                                     self.dy.to(DEV, BF16))
        assert torch.equal(got.cpu(), dx.to(torch.float32).to(BF16))


@pytest.mark.parametrize("rate", [0.0, 0.5])
@pytest.mark.parametrize("m,k,n,rank,group", [
    (100, 100, 33, 8, None), (90, 77, 41, 16, None), (1100, 96, 200, 4, 32), (70, 320, 17, 12, 20),
    (100, 100, 72, 40, None), (300, 77, 40, 64, None)])
def test_shapes_off_the_matrix_core_products(m, k, n, rank, group, rate):
    Exact(m, k, n, rank, group).check(rate)


# 256- and 192-column tiles of the large products, and the planners' own
@pytest.mark.parametrize("tile", [0, 18, 19])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 13, 16, 20, 24, 28, 32])
def test_ranks_in_the_large_products(tile, rank):
    with ops.tuning(int4_tile=tile, bf16_tile=tile):
        for rate in (0.0, 0.5):
            Exact(1100, 512, 456, rank, 64).check(rate)


def test_a_small_rank_at_sizes_that_take_the_large_products():
    Exact(4500, 2048, 2048, 4, 64).check(0.0)


@pytest.mark.parametrize("m", [1, 2, 13, 64, 100, 333])
@pytest.mark.parametrize("rank", [3, 16, 32])
def test_few_rows(m, rank):
    Exact(m, 256, 200, rank, 64).check(0.0)
    Exact(m, 2048, 2056, rank, 64).check(0.5)


@pytest.mark.parametrize("rank", [33, 40, 47, 48, 56, 64])
def test_ranks_above_32(rank):
    for m, k, n, group, tile in [(1100, 512, 456, 64, 0), (1100, 512, 456, 64, 18),
                                 (1100, 512, 456, 64, 19), (4500, 256, 264, None, 0),
                                 (100, 256, 33, 64, 0), (700, 1024, 2056, 32, 0)]:
        with ops.tuning(int4_tile=tile, bf16_tile=tile):
            for rate in (0.0, 0.5):
                Exact(m, k, n, rank, group).check(rate)


# every tile of packed weights (y) and of copied ones (dx) that has activation epilogues
@pytest.mark.parametrize("rank", [16, 32, 64])
@pytest.mark.parametrize("int4,bf16", [(1, 4), (2, 5), (3, 6), (10, 9), (11, 13), (12, 0), (17, 0)])
def test_every_tile(int4, bf16, rank):
    with ops.tuning(int4_tile=int4, bf16_tile=bf16):
        for rate in (0.0, 0.5):
            Exact(1100, 384, 392, rank, 64).check(rate)


def test_rank_64_at_sizes_that_take_the_large_products():
    Exact(4500, 2048, 2048, 64, 64).check(0.0)
