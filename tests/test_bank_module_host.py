"""Banks as modules: casts, precision policies, shared projections (CPU)."""

from __future__ import annotations

import copy

import pytest
import torch

import representax_amd as rx
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
