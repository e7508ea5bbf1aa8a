"""Banks as modules: casts, precision policies, shared projections (CPU)."""

from __future__ import annotations

import copy

import pytest
import torch

import representax_amd as rx
from representax_amd import bank as bank_module
from tests.test_bank_host import _adapter

BF16 = torch.bfloat16


@pytest.mark.parametrize("cast", [lambda m: m.to(BF16), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to(BF16).float(), lambda m: m.to("cpu", BF16),
                                  lambda m: copy.deepcopy(m).bfloat16()])
def test_scalings_stay_float32(cast):
    """alpha / r of 8 / 3 is no bf16 value: a cast would round it."""

    bank = rx.QuantizedLoRABank.from_adapters([_adapter(0, rank=3), _adapter(1, rank=3, alpha=1.0)])
    want = bank.scalings.clone()
    model = cast(torch.nn.Sequential(bank))
    assert model[0].scalings.dtype == torch.float32 and torch.equal(model[0].scalings, want)
    assert "scalings" in dict(model[0].named_buffers())
    assert torch.equal(model.state_dict()["0.scalings"], want)
    assert model.to("meta")[0].scalings.device.type == "meta"


@pytest.fixture
def taken(monkeypatch):
    """The types of A that banks call with, in the launch's place."""

    types = []

    def call(x, packed, scale_bits, lora_a, *rest, **options):
        types.append(lora_a.dtype)
        return x.new_zeros(*x.shape[:-1], packed.shape[0])

    monkeypatch.setattr(bank_module, "bank_linear", call)
    return types


def test_what_a_bank_computes_in(taken):
    bank = rx.QuantizedLoRABank.from_adapters([_adapter(0)])
    plan = rx.AdapterPlan(torch.empty(64, dtype=torch.uint8), 5, 1)
    x = torch.zeros(5, 64, dtype=BF16)
    policy = lambda config: rx.precision_context(rx.resolve_precision_policy(config))
    with rx.adapter_rows(plan):
        # the linear promotes these to float32
        with pytest.raises(TypeError, match="promoted to float32"):
            bank(x)
        with pytest.raises(TypeError, match="bfloat16"):
            bank(x.float())
        with rx.precision_context(rx.FP32_POLICY), pytest.raises(TypeError, match="bfloat16"):
            bank(x)
        assert not taken
        for config in (rx.PrecisionConfig.bfloat16_mixed(), rx.PrecisionConfig.float8_mixed()):
            with policy(config):
                assert bank(x).dtype == BF16 and bank(x.float()).dtype == BF16
        assert bank.to(BF16)(x).dtype == BF16
    assert taken == [torch.float32] * 4 + [BF16]


class _Pair(torch.nn.Module):
    def __init__(self, first, second):
        super().__init__()
        self.first, self.inner = first, torch.nn.ModuleList([second])


def test_an_adapter_in_two_places_is_one_bank():
    """Left where it was, the second place would serve every row the first model's adapter."""

    shared = [_adapter(i) for i in range(2)]
    banked = rx.bank_quantized_lora([_Pair(a, a) for a in shared])
    assert isinstance(banked.first, rx.QuantizedLoRABank) and banked.inner[0] is banked.first
    assert [torch.equal(banked.first.lora_a[i], a.lora_a) for i, a in enumerate(shared)] == [True] * 2
    # one model has it twice, the other two of them: two banks
    apart = rx.bank_quantized_lora([_Pair(shared[0], shared[0]), _Pair(shared[1], _adapter(5))])
    assert apart.inner[0] is not apart.first and [apart.first.site, apart.inner[0].site] == [0, 1]
    assert torch.equal(apart.inner[0].lora_a[1], _adapter(5).lora_a)
    with pytest.raises(ValueError, match="different places"):
        rx.bank_quantized_lora([_Pair(shared[0], shared[0]), _Pair(shared[1], torch.nn.GELU())])
