"""Hidden dropout in the BERT harness: rematerialized, captured, and off (GPU)."""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd.trainstep import BertConfig, MNRTrainStep, build_int4lora_encoder

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIG = dict(vocab_size=64, hidden_size=128, num_hidden_layers=2, num_attention_heads=2,
              intermediate_size=256, max_position_embeddings=32)


def _model(rate):
    model = build_int4lora_encoder(BertConfig(**CONFIG, hidden_dropout=rate), rank=8, alpha=16.0,
                                   device=DEV)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for p in rx.lora_parameters(model):
            p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    return model


def _gradients(model, remat, key):
    model.remat = remat
    ids = torch.arange(80, device=DEV).view(4, 20) % 64
    policy = rx.resolve_precision_policy(rx.PrecisionConfig.bfloat16_mixed())
    with rx.precision_context(policy):
        out = model.encode(ids, key=key)
    weight = torch.linspace(-1, 1, out.numel(), device=DEV).view(out.shape)
    return out.detach(), torch.autograd.grad((out * weight).sum(), rx.lora_parameters(model))


def test_a_rematerialized_layer_draws_the_same_masks():
    model = _model(0.2)
    key = rx.DropoutKeys(3, DEV).next()
    out, grads = _gradients(model, "none", key)
    again, regrads = _gradients(model, "full", key)
    assert torch.equal(out, again)
    for a, b in zip(grads, regrads):
        assert torch.equal(a, b)
    other, _ = _gradients(model, "none", rx.DropoutKeys(4, DEV).next())
    assert not torch.equal(out, other)


def test_without_a_key_or_training_nothing_is_dropped():
    key = rx.DropoutKeys(3, DEV).next()
    plain, _ = _gradients(_model(0.0), "none", None)
    dropped = _model(0.3)
    assert torch.equal(_gradients(dropped, "none", None)[0], plain)
    assert torch.equal(_gradients(dropped.eval(), "none", key)[0], plain)
    assert torch.equal(_gradients(_model(0.0), "none", key)[0], plain)


def test_a_captured_train_step_draws_a_new_key_each_replay():
    eager, captured = (MNRTrainStep(_model(0.1), batch=4, sequence=16) for _ in range(2))
    captured.capture(warmup=2)
    for _ in range(2):
        eager()
    for _ in range(3):
        a, b = eager().clone(), captured().clone()
        torch.cuda.synchronize()
        assert eager.keys.state.tolist() == captured.keys.state.tolist()
        # the same steps: the optimizer's own kernels may differ in a rounding
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(eager.flat, captured.flat, rtol=1e-4, atol=1e-6)


def test_a_captured_step_of_banks_with_every_dropout():
    """Adapters of two tasks in one batch, their dropout and the hidden one, layers run
    again in the backward: the captured step is the eager one, replay after replay, with
    eager work between."""

    index = torch.arange(8, device=DEV).repeat_interleave(16) % 3 - 1  # 4 queries, 4 documents
    plan = rx.adapter_plan(index, 2)
    key = torch.tensor([11, 0], device=DEV)
    steps = []
    for _ in range(2):
        models = [_model(0.1), _model(0.1)]
        with torch.no_grad():
            for p in rx.lora_parameters(models[1]):
                p.neg_()
        steps.append(MNRTrainStep(rx.bank_quantized_lora(models, dropout=0.2).train(), batch=4,
                                  sequence=16))
    eager, captured = steps
    with rx.adapter_rows(plan, key):
        captured.capture(warmup=2)
        for _ in range(2):
            eager()
    before, losses = captured.flat.detach().clone(), []
    for step in range(1, 4):
        key.copy_(torch.tensor([11, step], device=DEV))  # the adapters' masks of this step
        with rx.adapter_rows(plan, key):
            a = eager().clone()
        b = captured().clone()
        torch.cuda.synchronize()
        # the same steps: the optimizer's own kernels may differ in a rounding
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
        losses.append(float(b))
    assert len(set(losses)) == 3 and bool(captured.finite)
    torch.testing.assert_close(eager.flat, captured.flat, rtol=1e-4, atol=1e-6)
    assert not torch.equal(before, captured.flat)
