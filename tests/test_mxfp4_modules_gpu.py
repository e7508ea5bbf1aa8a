"""Hooks on MXFP4 projections see what separate calls would show them (GPU)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import representax_amd as rx
from tests.helpers import DEVICE

pytestmark = pytest.mark.gpu

POLICY = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())


def _linear(seed, rows, columns):
    return rx.Linear.init(columns, rows, key=seed, scale=columns ** -0.5, device=DEVICE)


def test_forward_and_backward_hooks_of_native_projections():
    gate, up, down = _linear(1, 96, 64), _linear(2, 96, 64), _linear(3, 64, 96)
    x = torch.randn((40, 64), device=DEVICE).to(torch.bfloat16)
    seen = []
    gate.register_forward_hook(lambda m, a, out: out * 2)
    up.register_full_backward_hook(lambda m, gin, gout: seen.append(gout[0].shape))
    with rx.precision_context(POLICY):
        y = rx.swiglu_mlp(x, gate, up, down)
        want = down(F.silu(gate(x)) * up(x))
    assert torch.equal(y, want)
    y.float().sum().backward()
    assert seen == [(40, 96)]


def test_forward_hooks_of_kept_projections():
    linears = [_linear(i, 96, 64) for i in (4, 5)]
    down = _linear(6, 64, 96)
    x = torch.randn((3, 64), device=DEVICE).to(torch.bfloat16)
    with rx.precision_context(POLICY), torch.no_grad():
        gate, up = (rx.MXFP4Linear.from_linear(l) for l in linears)
        up.register_forward_hook(lambda m, a, out: out + 1)
        assert torch.equal(rx.swiglu_mlp(x, gate, up, down), down(F.silu(gate(x)) * up(x)))
