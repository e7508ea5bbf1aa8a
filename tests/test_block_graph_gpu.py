"""Boundaries between blocks inside a graph: gradients that keep their graph, values that
change in place after the call (GPU)."""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd import ops

pytestmark = pytest.mark.gpu
DEV, F32, F64 = "cuda:0", torch.float32, torch.float64


def _parts():
    g = torch.Generator().manual_seed(2)
    draw = lambda *s: torch.randn(*s, generator=g)
    norm = rx.RMSNorm(64, 1e-6, DEV)
    with torch.no_grad():
        norm.weight.copy_(draw(64))
    return norm, draw(64, 64).to(DEV).requires_grad_(True), draw(3, 5, 64).to(DEV).requires_grad_(True)


def _layer(norm, w, x):
    """A block whose update and gate come from its stream, one norm before and after it."""

    return rx.block_norm(norm, x, torch.sin(x @ w), post=norm, gate=torch.tanh(x[:, :1] * 2),
                         scale=0.5, rate=0.25, key=torch.tensor([4, 2], device=DEV), site=1)


def _loss(out):
    return (out[0] ** 2).sum() + (out[1] ** 3).sum()


def test_gradients_that_keep_their_graph():
    """As the kernels' own and as the expressions' of 64 bits, and so are theirs. Sums of up
    to 64 float32 products over two nested norms: a hundred roundings of 2^-24 and their
    conditioning, far below 2^-12 of a gradient's norm."""

    norm, w, x = _parts()
    leaves = (x, w, norm.weight)
    plain = torch.autograd.grad(_loss(_layer(norm, w, x)), leaves)
    kept = torch.autograd.grad(_loss(_layer(norm, w, x)), leaves, create_graph=True)
    again = torch.autograd.grad(sum((v ** 2).sum() for v in kept), leaves)
    n64 = rx.RMSNorm(64, 1e-6, DEV).double()
    n64.load_state_dict(norm.state_dict())
    w64, x64 = (t.detach().to(F64).requires_grad_(True) for t in (w, x))
    leaves = (x64, w64, n64.weight)
    want = torch.autograd.grad(_loss(_layer(n64, w64, x64)), leaves, create_graph=True)
    want2 = torch.autograd.grad(sum((v ** 2).sum() for v in want), leaves)
    for a, b, c in zip(plain, kept, want):
        for v in (a, b):
            assert float((v.detach().to(F64) - c.detach()).norm() / c.detach().norm()) < 2.0 ** -12
    for a, b in zip(again, want2):
        assert float((a.to(F64) - b).norm() / b.norm()) < 2.0 ** -12


def test_the_stream_may_change_after_the_call():
    norm, w, x = _parts()
    want = torch.autograd.grad(_loss(rx.block_norm(norm, x * 1, x @ w)), (x, w))
    value = x * 1
    out = rx.block_norm(norm, value, x @ w)
    with torch.no_grad():
        value.add_(1)
    for a, b in zip(torch.autograd.grad(_loss(out), (x, w)), want):
        assert torch.equal(a, b)


def test_the_stream_is_not_kept():
    """Of a boundary the graph keeps t and the update, not the stream before it."""

    norm = rx.RMSNorm(2048, 1e-6, DEV)
    u = torch.randn(512, 2048, device=DEV, requires_grad=True)
    value = torch.randn_like(u).requires_grad_(True) * 1
    t, h = rx.block_norm(norm, value, u)
    before = torch.cuda.memory_allocated()
    size = value.numel() * 4
    del value
    assert before - torch.cuda.memory_allocated() >= size
    (t + h).sum().backward()
    assert u.grad is not None


def test_workspaces_are_released_and_made_again():
    norm, w, x = _parts()
    first = torch.autograd.grad(_loss(_layer(norm, w, x)), (x, w, norm.weight))
    stream = torch.cuda.current_stream()
    assert (x.get_device(), stream.cuda_stream) in ops._WORKSPACES
    stream.synchronize()
    ops.release_workspaces()
    assert not ops._WORKSPACES
    second = torch.autograd.grad(_loss(_layer(norm, w, x)), (x, w, norm.weight))
    assert ops._WORKSPACES and all(torch.equal(a, b) for a, b in zip(first, second))
