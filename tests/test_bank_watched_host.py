"""Banks where something watches the call: refused where a launch would be left out of
what is watched, and run where it would not (CPU, with the library's calls replaced)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import representax_amd as rx
from representax_amd import bank

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    """Launches that fill y with x's first column, on the CPU."""

    count = []

    def forward(x2d, a, b, packed, *rest):
        count.append(x2d.data_ptr())
        y = x2d[:, :1].detach().expand(-1, packed.shape[0]).contiguous()
        return y, (torch.zeros(len(x2d), 8, dtype=BF16) if rest[-1] else None)

    monkeypatch.setattr(bank, "_forward", forward)
    monkeypatch.setattr(bank, "_on_device", lambda *tensors: torch.device("cpu"))
    return count


def _call(x, **changed):
    args = dict(packed=torch.zeros(24, 32, dtype=torch.uint8),
                scale_bits=torch.zeros(24, dtype=torch.uint16), lora_a=torch.zeros(3, 8, 64),
                lora_b=torch.zeros(3, 24, 8), scalings=torch.ones(3),
                plan=rx.AdapterPlan(torch.empty(4096, dtype=torch.uint8), 5, 3))
    return rx.bank_linear(x, **(args | changed))


def test_forward_derivatives_are_refused(launches):
    x, a = torch.randn(5, 64).to(BF16), torch.zeros(3, 8, 64)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(x, lora_a=forward_ad.make_dual(a, torch.ones_like(a)))
        assert not launches
        # no operand has a tangent: the derivative is zero
        assert torch.equal(_call(x), x[:, :1].expand(-1, 24)) and len(launches) == 1


def test_traces_are_refused(launches):
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(_call, (torch.randn(5, 64).to(BF16),), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda i: rx.adapter_plan(i, 3).buffer,
                        (torch.zeros(5, dtype=torch.int32),), check_trace=False)
    assert not launches


def test_transforms_are_refused(launches):
    x = torch.randn(5, 64).to(BF16)
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.func.vmap(_call)(x.expand(2, 5, 64))
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.func.jvp(_call, (x,), (x,))
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.func.grad(lambda v: _call(v).sum())(x)
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.func.vmap(lambda i: rx.adapter_plan(i, 3).buffer)(torch.zeros(2, 5, dtype=torch.int32))
    assert not launches
    # closed over, it is a constant of the transform
    out = torch.func.vmap(lambda s: s * _call(x))(torch.ones(2, dtype=BF16))
    assert torch.equal(out[1], x[:, :1].expand(-1, 24))


def test_batched_gradients_are_refused(launches):
    x = torch.randn(5, 64).to(BF16).requires_grad_(True)
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.autograd.grad(_call(x), x, torch.ones(2, 5, 24, dtype=BF16), is_grads_batched=True)


def test_modes_and_compilers_meet_the_launch(launches):
    x = torch.randn(5, 64).to(BF16)
    want = x[:, :1].expand(-1, 24)
    with torch.device("cpu"):
        assert torch.equal(_call(x), want)
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):
        assert torch.equal(_call(x), want)
    compiled = torch.compile(_call, backend="eager")
    assert torch.equal(compiled(x), want)
    assert torch.equal(compiled(x.requires_grad_(True)).detach(), want)
    assert len(launches) == 4
