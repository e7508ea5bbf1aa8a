"""Dropout from a counter-based generator, whose mask is never stored (an
extension: the reference's encoders run without dropout).

The bits of a dropout are a function of a key (seed and step, int64, on the
device), of the call's ``site`` and of an element's place in the tensor's dense
order, so the backward, a rematerialized forward and a replayed graph make them
again. Element i has the 16 bits number i % 8 of Philox4x32-10 (Salmon et al.,
"Parallel random numbers: as easy as 1, 2, 3", 2011) for the counter (i / 8, its
high word, site, step); it is kept where they are below T = round(65536 (1 -
rate)), times 65536 / T, and zero otherwise.

Keys are values, as the reference's ``jax.random`` keys are: ``DropoutKeys.next``
gives a new one each step, and a step's calls differ in their ``site``.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _native as nat
from .ops import (BF16, F32, _aligned, _dtype_code, _stream, eager_calls, on_current_device,
                  plain_tensor)

_WORD = 0xFFFFFFFF
_KEY_SHAPE = torch.Size((2,))


class DropoutKeys(torch.nn.Module):
    """The keys of a run's steps: ``seed`` and a step counter on the device, so
    that ``next`` can be captured into a graph and each replay draws anew."""

    def __init__(self, seed: int, device=None) -> None:
        super().__init__()
        seed = int(seed) & 0x7FFFFFFFFFFFFFFF
        self.register_buffer("state", torch.tensor([seed, 0], dtype=torch.int64, device=device))

    @torch.no_grad()
    def next(self) -> torch.Tensor:
        """A new key: int64 ``[seed, step]``, step 1, 2, ..."""

        self.state[1:].add_(1)
        return self.state.clone()


def dropout_threshold(rate: float) -> int:
    """T of the given rate: 65536ths that are kept (at least one)."""

    return _threshold(float(rate))


@lru_cache(maxsize=256)
def _threshold(rate: float) -> int:
    if not 0.0 <= rate < 1.0:
        raise ValueError(f"dropout rate must be in [0, 1), got {rate}")
    return min(65536, max(1, round(65536 * (1.0 - rate))))


def check_key(key: torch.Tensor | None, site: int, device: torch.device) -> None:
    if key is None:
        raise ValueError("dropout needs a key (DropoutKeys.next)")
    if key.dtype != torch.int64 or key.shape != _KEY_SHAPE or key.device != device:
        raise ValueError(f"dropout key must be int64 [2] on {device}, got {key.dtype} "
                         f"{tuple(key.shape)} on {key.device}")
    if not 0 <= site <= _WORD:
        raise ValueError(f"dropout site must be 0 to 2^32 - 1, got {site}")


def kept(shape, key: torch.Tensor, threshold: int, site: int) -> torch.Tensor:
    """The mask itself, by torch operations: truth values of ``shape``."""

    count = torch.Size(shape).numel()
    block = torch.arange(-(-count // 8), dtype=torch.int64, device=key.device)
    c = [block & _WORD, block >> 32, torch.full_like(block, int(site)),
         (key[1] & _WORD).expand_as(block)]
    k = [key[0] & _WORD, (key[0] >> 32) & _WORD]
    for _ in range(10):
        # products of 32-bit words in 64 bits: the bits are right though the sign is not
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & _WORD) ^ c[1] ^ k[0], b & _WORD, ((a >> 32) & _WORD) ^ c[3] ^ k[1],
             a & _WORD]
        k = [(k[0] + 0x9E3779B9) & _WORD, (k[1] + 0xBB67AE85) & _WORD]
    words = torch.stack(c, 1)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:count]
    return (bits < threshold).reshape(shape)


def dropped(value: torch.Tensor, key: torch.Tensor, threshold: int, site: int) -> torch.Tensor:
    """The torch expression of a dropout, in the value's type."""

    if threshold == 65536:
        return value
    keep = kept(value.shape, key, threshold, site)
    return torch.where(keep, value * (65536.0 / threshold), torch.zeros_like(value))


def _wide(dtype: torch.dtype) -> torch.dtype:
    return torch.promote_types(dtype, F32)


def _launch(x, key, threshold, site):
    x = _aligned(x)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    args = (x.data_ptr(), _dtype_code(x.dtype), x.numel(), key.data_ptr(), site, threshold,
            out.data_ptr(), _stream(x.device))
    binding = nat.fast()
    if binding is not None:
        nat.check(binding.dropout(*args))
    else:
        nat.call("rpx_dropout", *args)
    return out


class DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, key, rate, threshold, site):
        ctx.save_for_backward(key)
        ctx.args = (rate, threshold, site)
        return _launch(x, key, threshold, site)

    @staticmethod
    def backward(ctx, grad):
        (key,) = ctx.saved_tensors
        rate, threshold, site = ctx.args
        if (not torch.is_grad_enabled() and eager_calls() and plain_tensor(grad)
                and on_current_device(grad)):
            return _launch(grad, key, threshold, site), None, None, None, None
        return dropout(grad, rate, key, site), None, None, None, None


def dropout(value: torch.Tensor, rate: float, key: torch.Tensor, site: int = 0) -> torch.Tensor:
    """``value`` with a share ``rate`` of its elements zero and the others scaled
    up, the mask drawn from ``key`` and ``site``; differentiable. bf16 and float32
    device tensors in one pass over memory, anything else by torch operations.
    A dropped element is zero whatever its value was."""

    threshold = dropout_threshold(rate)
    if not value.is_floating_point():
        raise TypeError(f"dropout takes floating-point values, got {value.dtype}")
    if threshold == 65536:
        return value
    check_key(key, site, value.device)
    if (eager_calls() and plain_tensor(value) and plain_tensor(key) and on_current_device(value)
            and value.dtype in (BF16, F32) and value.layout == torch.strided):
        key = key.contiguous()
        if torch.is_grad_enabled() and value.requires_grad:
            return DropoutFn.apply(value, key, rate, threshold, int(site))
        return _launch(value, key, threshold, int(site))
    return dropped(value.to(_wide(value.dtype)), key, threshold, int(site)).to(value.dtype)


__all__ = ["DropoutKeys", "dropout"]
