"""MXFP4 modules on the host: which projections ``swiglu_mlp`` calls and which it runs
in one kernel, and which calls refuse gradients (CPU only, nothing launched)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import representax_amd as rx
from oracle import mxfp4 as omx

POLICY = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())


class Scaled(rx.Linear):
    """A projection with a forward of its own, which runs on any device."""

    def forward(self, value):
        return 3.0 * F.linear(value, self.weight.to(value.dtype))


class Kept(rx.MXFP4Linear):
    def forward(self, value):
        return torch.ones((*value.shape[:-1], self.output_size), dtype=value.dtype)


def _linears(cls, *shapes):
    g = torch.Generator().manual_seed(1)
    return [cls(torch.randn(s, generator=g)) for s in shapes]


def _kept(rows, columns, cls=rx.MXFP4Linear):
    codes, scales = omx.stored(torch.ones((rows, columns)).numpy())
    return cls(rx.MXFP4Matrix(torch.from_numpy(codes), torch.from_numpy(scales), columns))


def test_projections_of_a_subclass_run_their_own_forward():
    x = torch.randn(3, 4, 8).to(torch.bfloat16)
    gate, up, down = _linears(Scaled, (6, 8), (6, 8), (8, 6))
    want = down(F.silu(gate(x)) * up(x))
    with rx.precision_context(POLICY):
        assert torch.equal(rx.swiglu_mlp(x, gate, up, down), want)
        kept = [_kept(6, 8, Kept) for _ in range(2)]
        want = down(F.silu(torch.ones(3, 4, 6)).to(torch.bfloat16))
        assert torch.equal(rx.swiglu_mlp(x, *kept, down), want)


def test_a_replaced_forward_runs():
    x = torch.randn(5, 8).to(torch.bfloat16)
    gate, up, down = _linears(rx.Linear, (6, 8), (6, 8), (8, 6))
    for module in (gate, up, down):
        module.forward = lambda v, w=module.weight: F.linear(v, w.detach().to(v.dtype))
    want = down(F.silu(gate(x)) * up(x))
    with rx.precision_context(POLICY):
        assert torch.equal(rx.swiglu_mlp(x, gate, up, down), want)


@pytest.mark.parametrize("make", [lambda: _linears(rx.Linear, (6, 8))[0], lambda: _kept(6, 8)])
@pytest.mark.parametrize("register", ["register_forward_pre_hook", "register_forward_hook",
                                      "register_full_backward_pre_hook",
                                      "register_full_backward_hook"])
@pytest.mark.parametrize("hooked", [0, 1])
def test_hooked_projections_are_called(make, register, hooked, monkeypatch):
    """A projection with a hook of any kind is called, and so is its neighbour."""

    x = torch.randn(5, 8).to(torch.bfloat16)
    pair = [make(), make()]
    getattr(pair[hooked], register)(lambda *a: None)
    called = []
    for cls in (rx.Linear, rx.MXFP4Linear):
        monkeypatch.setattr(cls, "forward", lambda self, value: (
            called.append(self), value[:, :6] * 2.0)[1])
    with rx.precision_context(POLICY):
        y = rx.swiglu_mlp(x, *pair, torch.nn.Identity())
    assert called == pair
    assert torch.equal(y, F.silu(x[:, :6] * 2.0) * (x[:, :6] * 2.0))


def test_projections_without_hooks_stay_in_one_kernel(monkeypatch):
    """Neither is called: the fused entry is reached, which takes device tensors only."""

    x = torch.randn(5, 8).to(torch.bfloat16)
    for cls in (rx.Linear, rx.MXFP4Linear):
        monkeypatch.setattr(cls, "forward", lambda self, value: pytest.fail("called"))
    for pair in (_linears(rx.Linear, (6, 8), (6, 8)), [_kept(6, 8), _kept(6, 8)]):
        with rx.precision_context(POLICY), pytest.raises(RuntimeError, match="ROCm"):
            rx.swiglu_mlp(x, *pair, torch.nn.Identity())


def test_kept_weights_refuse_a_gradient():
    """Their results would be cut off from the graph without a word."""

    x = torch.randn(5, 8).to(torch.bfloat16).requires_grad_()
    module = _kept(6, 8)
    calls = [lambda v: rx.mxfp4_linear(v, module.weight),
             lambda v: rx.mxfp4_gated(v, module.weight, module.weight), module,
             lambda v: rx.swiglu_mlp(v, module, module, torch.nn.Identity())]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradients"):
            call(x)
        with pytest.raises(RuntimeError, match="no gradients"):
            call(x * 2)  # no leaf
        # no gradient is wanted: refused only for the device
        with pytest.raises(RuntimeError, match="ROCm"):
            call(x.detach())
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm"):
            call(x)
