"""The boundary between two blocks by torch operations, and refusals (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.nn.functional as F

import representax_amd as rx
from representax_amd import _native as nat
from representax_amd.philox import dropped
from representax_amd.norms import _rows_per_gate

F64 = torch.float64


def _norms(kind, size):
    g = torch.Generator().manual_seed(size)
    cls = rx.LayerNorm if kind == "layer" else rx.RMSNorm
    norm = cls(size, 1e-6).double()
    with torch.no_grad():
        for p in norm.parameters():
            p.copy_(torch.randn(size, generator=g, dtype=F64))
    return norm


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", [None, (12,), (2, 1, 12), (2, 3, 12), (3, 12)])
def test_expression_and_its_gradients(kind, gate):
    norm, post = _norms(kind, 12), _norms("rms", 12)
    x, u = (torch.randn(2, 3, 12, dtype=F64, requires_grad=True) for _ in range(2))
    gate = None if gate is None else torch.randn(gate, dtype=F64, requires_grad=True)
    key = torch.tensor([4, 2])

    def call(x, u, *more):
        return rx.block_norm(norm, x, u, post=post, gate=more[0] if more else None, scale=0.5,
                             rate=0.25, key=key, site=3)

    leaves = (x, u) if gate is None else (x, u, gate)
    p = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + 1e-6) * post.weight
    p = p if gate is None else p * gate
    t = x + 0.5 * dropped(p, key, 49152, 3)
    got_t, got_h = call(*leaves)
    torch.testing.assert_close(got_t, t)
    want = (F.layer_norm(t, (12,), norm.weight, norm.bias, 1e-6) if kind == "layer"
            else t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * norm.weight)
    torch.testing.assert_close(got_h, want)
    assert torch.autograd.gradcheck(call, leaves)


def test_a_plain_call_is_add_norm():
    norm = _norms("rms", 8).float()
    x, u = torch.randn(5, 8), torch.randn(5, 8)
    for got, want in zip(rx.block_norm(norm, x, u), rx.add_norm(norm, x, u)):
        torch.testing.assert_close(got, want)
    t, h = rx.block_norm(None, x, u, scale=2.0)
    torch.testing.assert_close(t, x + 2 * u)
    assert h is None


def test_other_modules_are_called():
    class Twice(torch.nn.Module):
        def forward(self, v):
            return 2 * v

    x, u = torch.randn(3, 8), torch.randn(3, 8)
    t, h = rx.block_norm(Twice(), x, u, post=Twice())
    torch.testing.assert_close(t, x + 2 * u)
    torch.testing.assert_close(h, 2 * t)


@pytest.mark.parametrize("gate,shape,want", [
    ((8,), (4, 6, 8), 24), ((1, 1, 8), (4, 6, 8), 24), ((4, 1, 8), (4, 6, 8), 6),
    ((4, 6, 8), (4, 6, 8), 1), ((6, 8), (4, 6, 8), None), ((1, 6, 8), (4, 6, 8), None),
    ((4, 6, 1), (4, 6, 8), None), ((1, 8), (1, 8), 1), ((1, 1, 8), (1, 6, 8), 6)])
def test_rows_per_gate(gate, shape, want):
    assert _rows_per_gate(torch.empty(gate), shape) == want


def test_refusals():
    norm = rx.RMSNorm(8, 1e-6)
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="shape"):
        rx.block_norm(norm, x, x[:2])
    with pytest.raises(ValueError, match="gate"):
        rx.block_norm(norm, x, x, gate=torch.ones(3, 4, 8))
    with pytest.raises(ValueError, match="key"):
        rx.block_norm(norm, x, x, rate=0.1)
    with pytest.raises(ValueError, match="rate"):
        rx.block_norm(norm, x, x, rate=1.0, key=torch.zeros(2, dtype=torch.int64))


def _block(**fields):
    p = 1 << 20
    norm = nat.BlockNorm(p, p, nat.DTYPE_BF16, nat.NORM_LAYER, 1e-6)
    values = dict(x=p, u=p, gate=None, rows_per_gate=1, post=nat.BlockNorm(), norm=norm, key=p,
                  site=0, threshold=65536, rows=4, size=8, t=p, h=p, dtype=nat.DTYPE_BF16,
                  gate_dtype=nat.DTYPE_BF16, scale=1.0)
    values.update(fields)
    return nat.Block(**values)


@pytest.mark.parametrize("fields,match", [
    ({"dtype": 5}, "dtype"), ({"rows": -1}, "rows"), ({"size": 0}, "size"),
    ({"size": 8193}, "size"), ({"gate": 1 << 20, "rows_per_gate": 3}, "rows_per_gate"),
    ({"gate": 1 << 20, "rows_per_gate": 0}, "rows_per_gate"), ({"threshold": 0}, "threshold"),
    ({"threshold": 5, "key": None}, "key"), ({"site": -1}, "site"), ({"x": None}, "null"),
    ({"h": None}, "null"), ({"x": 3}, "aligned"),
    ({"norm": nat.BlockNorm(16, None, 1, nat.NORM_LAYER, 0.1)}, "bias"),
    ({"norm": nat.BlockNorm(16, 16, 1, 7, 0.1)}, "kind"),
    ({"post": nat.BlockNorm(16, 16, 7, 0, 0.1)}, "dtype")])
def test_forward_entry_point_refuses(fields, match):
    with pytest.raises(ValueError, match=match):
        nat.call("rpx_block_forward", ctypes.byref(_block(**fields)), None)


def test_backward_entry_point_refuses():
    p = 1 << 20

    def call(grads, ws=None, nbytes=0, **fields):
        nat.call("rpx_block_backward", ctypes.byref(_block(**fields)),
                 ctypes.byref(nat.BlockGradients(**grads)), ws, nbytes, None)

    for grads, match in [({"d_gate": p}, "does not have"), ({"d_post_weight": p}, "does not have"),
                         ({"dh": p, "d_weight": p}, "workspace"), ({"dh": 3}, "aligned")]:
        with pytest.raises(ValueError, match=match):
            call(grads)
    with pytest.raises(ValueError, match="without its norm"):
        call({"dh": p}, norm=nat.BlockNorm())
    with pytest.raises(ValueError, match="no rows"):
        call({"d_weight": p}, rows=0)
    assert nat.query("rpx_block_backward_workspace", ctypes.byref(_block(size=9000)),
                     ctypes.byref(nat.BlockGradients())) == 0
