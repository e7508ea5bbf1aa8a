"""Banks of adapters: what is refused, and how they are put together (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import representax_amd as rx
from representax_amd import _native as nat
from representax_amd.bank import active_adapter_rows

BF16 = torch.bfloat16


def _operands(k=64, n=24, e=3, r=8):
    return dict(packed=torch.zeros(n, k // 2, dtype=torch.uint8),
                scale_bits=torch.zeros(n, dtype=torch.uint16),
                lora_a=torch.zeros(e, r, k), lora_b=torch.zeros(e, n, r), scalings=torch.ones(e),
                plan=rx.AdapterPlan(torch.empty(4096, dtype=torch.uint8), 5, e))


def _adapter(seed, rank=4, n=24, k=64, alpha=8.0, base=0, group=None):
    g = torch.Generator().manual_seed(base)
    bits = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.int32).to(torch.uint8)
    h = torch.Generator().manual_seed(seed + 100)
    return rx.QuantizedLoRALinear(
        packed_weight=bits(n, k // 2), scale_bits=torch.ones(n, dtype=BF16).view(torch.uint16),
        bias_bits=None, lora_a=torch.randn(rank, k, generator=h),
        lora_b=torch.randn(n, rank, generator=h), input_size=k, output_size=n, rank=rank,
        alpha=alpha, group_size=group)


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(5, 64)), TypeError, "bfloat16 activations"),
    (dict(x=torch.zeros(5, 62, dtype=BF16)), ValueError, "packed"),
    (dict(packed=torch.zeros(24, 32, dtype=torch.int8)), ValueError, "packed"),
    (dict(scale_bits=torch.zeros(23, dtype=torch.uint16)), ValueError, "scale_bits"),
    (dict(group_size=3), ValueError, "group_size"),
    (dict(group_size=-2), ValueError, "group_size"),
    (dict(lora_a=torch.zeros(3, 8, 63)), ValueError, "lora_a"),
    (dict(lora_a=torch.zeros(8, 64)), ValueError, "lora_a"),
    (dict(lora_b=torch.zeros(3, 24, 7)), ValueError, "lora_b"),
    (dict(scalings=torch.ones(2)), ValueError, "scalings"),
    (dict(scalings=torch.ones(3, dtype=torch.float64)), TypeError, "scalings"),
    (dict(lora_a=torch.zeros(3, 8, 64, dtype=torch.float16)), TypeError, "lora_a"),
    (dict(lora_a=torch.zeros(3, 65, 64), lora_b=torch.zeros(3, 24, 65)), ValueError, "rank"),
    (dict(bias=torch.zeros(23, dtype=BF16)), ValueError, "bias"),
    (dict(x=torch.zeros(4, 64, dtype=BF16)), ValueError, "plan"),
    (dict(plan=rx.AdapterPlan(torch.empty(9), 5, 4)), ValueError, "plan"),
    (dict(rate=1.0), ValueError, "rate"), (dict(rate=0.5), ValueError, "key"),
    (dict(), RuntimeError, "ROCm devices only")])
def test_bank_linear_refuses(change, error, match):
    args = {"x": torch.zeros(5, 64, dtype=BF16), **_operands()} | change
    with pytest.raises(error, match=match):
        rx.bank_linear(**args)


@pytest.mark.parametrize("index,adapters,error", [
    ([0, 1, 3], 3, ValueError), ([-2, 0], 3, ValueError), ([0], 0, ValueError),
    ([0], 1025, ValueError), (torch.zeros(3), 3, TypeError), ([0.5], 3, TypeError),
    (torch.zeros(3, dtype=torch.int16), 3, TypeError)])
def test_plans_refuse(index, adapters, error):
    with pytest.raises(error):
        rx.adapter_plan(index, adapters)


def _bank(**fields):
    p = 1 << 20
    values = dict(x=p, m=5, k=64, packed=p, scale_bits=p, n=24, group_size=0, bias_bits=None,
                  lora_a=p, lora_b=p, scalings=p, adapters=3, rank=8, plan=p, plan_bytes=1 << 20,
                  key=None, site=0, threshold=65536)
    values.update(fields)
    return nat.Bank(**values)


@pytest.mark.parametrize("fields,match", [
    ({"m": -1}, "rows"), ({"m": (1 << 25) + 1}, "rows"), ({"adapters": 0}, "adapters"),
    ({"adapters": 1025}, "adapters"), ({"rank": 0}, "rank"), ({"rank": 65}, "rank"),
    ({"n": 0}, "n >= 1"), ({"k": 1 << 23}, "2\\^23"), ({"group_size": 24}, "group_size"),
    ({"threshold": 0}, "threshold"), ({"threshold": 9}, "key"), ({"site": 1 << 32}, "site"),
    ({"x": None}, "null"), ({"plan": None}, "null"), ({"lora_b": (1 << 20) + 2}, "aligned"),
    ({"scalings": (1 << 20) + 2}, "aligned"), ({"plan_bytes": 16}, "plan")])
def test_entry_points_refuse(fields, match):
    p = ctypes.c_void_p(1 << 20)
    bank = _bank(**fields)
    with pytest.raises(ValueError, match=match):
        nat.call("rpx_bank_forward", ctypes.byref(bank), p, None, p, 1 << 30, None)
    with pytest.raises(ValueError, match=match):
        nat.call("rpx_bank_backward", ctypes.byref(bank), p, p, p, p, 0, p, 0, p, 1 << 30, None)
    assert nat.query("rpx_bank_forward_workspace", ctypes.byref(bank), 0) == 0


def test_outputs_and_workspaces_are_checked():
    p = ctypes.c_void_p(1 << 20)
    big = _bank(m=500)
    ref = ctypes.byref(big)
    assert nat.query("rpx_bank_forward_workspace", ref, 0) > 0
    for args, match in [((None, None, p, 1 << 30), "null"),
                        ((ctypes.c_void_p(24), None, p, 1 << 30), "aligned"),
                        ((p, None, None, 0), "workspace")]:
        with pytest.raises(ValueError, match=match):
            nat.call("rpx_bank_forward", ref, *args, None)
    with pytest.raises(ValueError, match="dtype"):
        nat.call("rpx_bank_backward", ref, p, p, p, p, 3, p, 0, p, 1 << 30, None)
    with pytest.raises(ValueError, match="workspace"):
        nat.call("rpx_bank_backward", ref, p, p, p, p, 0, p, 0, None, 0, None)
    nat.call("rpx_bank_forward", ctypes.byref(_bank(m=0)), None, None, None, 0, None)
    with pytest.raises(ValueError, match="index"):
        nat.call("rpx_adapter_plan", p, 2, 5, 3, p, 1 << 20, None)
    with pytest.raises(ValueError, match="too small"):
        nat.call("rpx_adapter_plan", p, 4, 5, 3, p, 8, None)
    with pytest.raises(ValueError, match="aligned"):
        nat.call("rpx_adapter_plan", ctypes.c_void_p(20), 8, 5, 3, p, 1 << 20, None)


def test_from_adapters_pads_ranks_and_takes_one_back():
    adapters = [_adapter(0, rank=4), _adapter(1, rank=2, alpha=3.0)]
    bank = rx.QuantizedLoRABank.from_adapters(adapters, dropout=0.1, site=4)
    assert bank.lora_a.shape == (2, 4, 64) and bank.lora_b.shape == (2, 24, 4)
    assert torch.equal(bank.lora_a[1, :2], adapters[1].lora_a) and not bank.lora_a[1, 2:].any()
    assert not bank.lora_b[1, :, 2:].any()
    assert bank.scalings.tolist() == [2.0, 1.5]
    one = bank.adapter(1)
    assert one.scaling == 1.5 and torch.equal(one.lora_b, bank.lora_b[1])
    assert rx.lora_parameter_filter(bank) == {"lora_a": True, "lora_b": True}


def test_banks_need_one_base():
    with pytest.raises(ValueError, match="one base"):
        rx.QuantizedLoRABank.from_adapters([_adapter(0), _adapter(1, base=1)])
    with pytest.raises(ValueError, match="at least one"):
        rx.QuantizedLoRABank.from_adapters([])
    with pytest.raises(ValueError, match="rate"):
        rx.QuantizedLoRABank.from_adapters([_adapter(0)], dropout=1.0)


def test_models_of_one_base_become_one():
    models = [torch.nn.Sequential(_adapter(i), torch.nn.GELU(), _adapter(i + 7, n=64)).eval()
              for i in range(3)]
    banked = rx.bank_quantized_lora(models)
    banks = [m for m in banked.modules() if isinstance(m, rx.QuantizedLoRABank)]
    assert [b.site for b in banks] == [0, 1] and not any(b.training for b in banks)
    for i, model in enumerate(models):
        assert torch.equal(banked[2].lora_a[i], model[2].lora_a)
    with pytest.raises(ValueError, match="different places"):
        rx.bank_quantized_lora([models[0], torch.nn.Sequential(models[1][0])])
    with pytest.raises(ValueError, match="no QuantizedLoRALinear"):
        rx.bank_quantized_lora([torch.nn.GELU()])


def test_a_bank_is_called_under_its_rows():
    bank = rx.QuantizedLoRABank.from_adapters([_adapter(0)])
    with pytest.raises(RuntimeError, match="adapter_rows"):
        bank(torch.zeros(5, 64, dtype=BF16))
    plan = rx.AdapterPlan(torch.empty(64, dtype=torch.uint8), 5, 1)
    with rx.adapter_rows(plan):
        assert active_adapter_rows() == (plan, None)
        with pytest.raises(TypeError, match="bfloat16"):
            bank(torch.zeros(5, 64))
    assert active_adapter_rows() is None
