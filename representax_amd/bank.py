"""Low-rank adapters of many requests beside one packed INT4 projection.

A bank holds several adapters over one frozen base; every row of a batch names
its own (or none). ``adapter_plan`` sorts a batch's rows by adapter once, for
every projection that the batch goes through, and ``bank_linear`` is one
projection: ``y[i] = x[i] W_b^T + bias + s_e (dropout(x[i]) A_e^T) B_e^T`` with
``e = index[i]``, QuantizedLoRALinear's forward
(src/representax/models/adapters.py:158-182) for each row. Serving: requests of
many tenants or tasks in one batch, down to one token. Training: several
adapters at once, with the gradients of x, A and B.

``QuantizedLoRABank`` is the module, ``bank_quantized_lora`` puts banks in the
place of the adapters of several models over one base, and ``adapter_rows`` says
which adapter each row of the calls inside it takes.

The arithmetic is bf16 products with float32 sums and one rounding of y and of dx;
h and its gradient are rounded to bf16 where they are operands of matrix products
(for few rows, y takes h as float32 sums).
"""

from __future__ import annotations

import copy
import ctypes
from contextlib import contextmanager, nullcontext
from contextvars import ContextVar
from typing import Iterator, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat
from .adapters import QuantizedLoRALinear, _set_module
from .philox import check_key, dropout_threshold
from .ops import (BF16, F32, _aligned, _as, _check_extent, _dtype_code, _has_storage, _on_device,
                  _ptr, _stream, _u16, _workspace, cast_many, eager_calls, group_arg,
                  on_current_device)
from .precision import (active_compute_dtype, activation_inputs, compute_operands,
                        compute_parameter_dtype)
from .sharding import constrain_activation

MAX_ADAPTERS = 1024
MAX_RANK = 64
MAX_ROWS = 1 << 25


_HERE = nullcontext()


def _on(device: torch.device, t: torch.Tensor):
    """Launches go to the current device: make it the tensors'."""

    return _HERE if on_current_device(t) else torch.cuda.device(device)


def _check_unwatched(what: str, *tensors: torch.Tensor | None) -> None:
    """A launch is in no trace, and has no batching rule and no forward derivative: where
    one of them is asked for, it is refused rather than left out."""

    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{what} cannot be traced")
    for t in tensors:
        if t is None:
            continue
        if not _has_storage(t):
            raise RuntimeError(f"{what} takes no tensors of function transforms (vmap, jvp, grad)")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


class AdapterPlan:
    """The rows of a batch sorted by adapter (``adapter_plan``): good for every
    projection of the batch, and for later batches with the same index."""

    def __init__(self, buffer: torch.Tensor, rows: int, adapters: int) -> None:
        self.buffer = buffer
        self.rows = rows
        self.adapters = adapters


def adapter_plan(index, adapters: int, device=None) -> AdapterPlan:
    """The plan of a batch whose row i takes adapter ``index[i]`` of ``adapters``,
    or none where it is -1.

    ``index``: an int32 or int64 tensor (any shape, rows in its dense order), or
    numbers. On the host it is checked here and copied to ``device`` (default: the
    current one). On the device nothing is waited for: an entry outside the bank
    counts as -1, and ``ops.check_device_errors`` reports it. One small launch, which
    a graph may capture: a replay reads the index anew."""

    adapters = int(adapters)
    if not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"a bank has 1 to {MAX_ADAPTERS} adapters, got {adapters}")
    if not isinstance(index, torch.Tensor):
        index = torch.as_tensor(index)
        index = index.to(torch.int32) if index.numel() == 0 else index
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"adapter index must be int32 or int64, got {index.dtype}")
    if not eager_calls():
        _check_unwatched("adapter_plan", index)
    if index.numel() > MAX_ROWS:
        raise ValueError(f"a plan has at most {MAX_ROWS} rows, got {index.numel()}")
    if not index.is_cuda:
        if index.numel() and not -1 <= int(index.min()) <= int(index.max()) < adapters:
            raise ValueError(f"adapter index must be -1 to {adapters - 1}")
        index = index.to(torch.device("cuda") if device is None else device)
    rows = index.numel()
    device = _on_device(index)
    index = index.contiguous()
    nbytes = nat.query("rpx_adapter_plan_bytes", rows, adapters)
    buffer = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _on(device, index):
        nat.call("rpx_adapter_plan", _ptr(index), index.element_size(), rows, adapters,
                 _ptr(buffer), nbytes, _stream(device))
    return AdapterPlan(buffer, rows, adapters)


def _bank_fields(x2d, packed, scale_bits, bias, a, b, scalings, plan, key, cfg):
    """The fields of an ``rpx_bank``."""

    m, k = x2d.shape
    e, r, _ = a.shape
    return (x2d.data_ptr(), m, k, packed.data_ptr(), scale_bits.data_ptr(), packed.shape[0],
            cfg["group"], _ptr(bias), a.data_ptr(), b.data_ptr(), scalings.data_ptr(), e, r,
            plan.data_ptr(), plan.numel(), _ptr(key), cfg["site"], cfg["threshold"])


def _forward(x2d, a, b, packed, scale_bits, bias, scalings, plan, key, cfg, need_h):
    device = x2d.device
    fields = _bank_fields(x2d, packed, scale_bits, bias, a, b, scalings, plan, key, cfg)
    m = x2d.shape[0]
    y = torch.empty((m, packed.shape[0]), dtype=BF16, device=device)
    h = None
    if need_h:
        h = torch.empty((m, -(-a.shape[1] // 8) * 8), dtype=BF16, device=device)
    with _on(device, x2d):
        stream = _stream(device)
        nbytes = nat.bank_call("forward_workspace", fields, int(need_h))
        ws = _workspace(nbytes, device, stream) if nbytes else None
        nat.bank_call("forward", fields, y.data_ptr(), _ptr(h), _ptr(ws), nbytes, stream)
    return y, h


class BankLinearFn(torch.autograd.Function):
    """Autograd node of ``bank_linear`` on 2-D activations; A and B are the masters
    or their compute views, and get gradients in their type."""

    @staticmethod
    def forward(ctx, x2d, lora_a, lora_b, packed, scale_bits, bias, scalings, plan, key, cfg):
        a, b = (_aligned(t) for t in cast_many((lora_a, lora_b), BF16))
        y, h = _forward(x2d, a, b, packed, scale_bits, bias, scalings, plan, key, cfg, True)
        ctx.save_for_backward(x2d, a, b, packed, scale_bits, scalings, plan, key, h)
        ctx.cfg, ctx.dtypes = cfg, (lora_a.dtype, lora_b.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x2d, a, b, packed, scale_bits, scalings, plan, key, h = ctx.saved_tensors
        need_x, need_a, need_b = ctx.needs_input_grad[:3]
        if not eager_calls() or not _has_storage(grad):
            _check_unwatched("the gradient of bank_linear", grad)
        grad = _aligned(_as(grad, BF16))
        device = _on_device(grad, x2d)
        fields = _bank_fields(x2d, packed, scale_bits, None, a, b, scalings, plan, key, ctx.cfg)
        dx = torch.empty_like(x2d) if need_x else None
        d_a = torch.empty(a.shape, dtype=ctx.dtypes[0], device=device) if need_a else None
        d_b = torch.empty(b.shape, dtype=ctx.dtypes[1], device=device) if need_b else None
        with _on(device, x2d):
            stream = _stream(device)
            nbytes = nat.bank_call("backward_workspace", fields, need_x, need_a, need_b)
            ws = _workspace(nbytes, device, stream) if nbytes else None
            nat.bank_call("backward", fields, grad.data_ptr(), h.data_ptr(), _ptr(dx), _ptr(d_a),
                          _dtype_code(ctx.dtypes[0]), _ptr(d_b), _dtype_code(ctx.dtypes[1]),
                          _ptr(ws), nbytes, stream)
        return dx, d_a, d_b, None, None, None, None, None, None, None


def _check_bank(k, packed, scale_bits, lora_a, lora_b, scalings, group_size, bias):
    if packed.dtype != torch.uint8 or packed.dim() != 2 or packed.shape[1] != (k + 1) // 2:
        raise ValueError(f"packed weight must be uint8 [N, {(k + 1) // 2}], got {packed.dtype} "
                         f"{tuple(packed.shape)}")
    n = packed.shape[0]
    g = group_arg(group_size, k)
    if g and (g < 0 or k % g or g % 2):
        raise ValueError(f"group_size must be even and divide the input size {k}, got {g}")
    if scale_bits.numel() != n * (k // g if g else 1):
        raise ValueError(f"scale_bits: {tuple(scale_bits.shape)} for {n} rows of {k} columns in "
                         f"groups of {g or k}")
    if lora_a.dim() != 3 or lora_a.shape[2] != k:
        raise ValueError(f"lora_a: shape {tuple(lora_a.shape)}, expected (adapters, rank, {k})")
    e, r, _ = lora_a.shape
    _check_extent("lora_b", lora_b, (e, n, r))
    _check_extent("scalings", scalings, (e,))
    if not 1 <= e <= MAX_ADAPTERS or not 1 <= r <= MAX_RANK:
        raise ValueError(f"a bank has 1 to {MAX_ADAPTERS} adapters of rank 1 to {MAX_RANK}, got "
                         f"{e} of rank {r}")
    for name, t in (("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype not in (BF16, F32):
            raise TypeError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if scalings.dtype != F32:
        raise TypeError(f"scalings must be float32, got {scalings.dtype}")
    if bias is not None and bias.numel() != n:
        raise ValueError(f"bias: shape {tuple(bias.shape)}, expected ({n},)")
    return n, e, r


def bank_linear(x: torch.Tensor, packed: torch.Tensor, scale_bits: torch.Tensor,
                lora_a: torch.Tensor, lora_b: torch.Tensor, scalings: torch.Tensor,
                plan: AdapterPlan, *, group_size: int | None = None,
                bias: torch.Tensor | None = None, rate: float = 0.0,
                key: torch.Tensor | None = None, site: int = 0) -> torch.Tensor:
    """``x [..., K] -> y [..., N]`` over one INT4 projection (``packed``,
    ``scale_bits``, ``group_size`` and ``bias``, bf16 or its bits, as
    ``QuantizedLoRALinear`` keeps them), row i with the adapter that ``plan`` gives
    it: ``lora_a [E, r, K]``, ``lora_b [E, N, r]`` (float32 masters or bf16 views)
    and ``scalings [E]`` (float32, alpha / r). ``rate``, ``key`` and ``site``: dropout
    of the adapters' input, as ``dropout(x, rate, key, site)`` draws it.

    bf16 activations; gradients reach x, A and B (once: there is no second
    derivative). Adapters without rows get gradients of zero. One adapter's values
    never reach another's rows. Traces, function transforms (``torch.func``) and
    forward-mode derivatives are refused."""

    if not eager_calls():
        _check_unwatched("bank_linear", x, packed, scale_bits, lora_a, lora_b, scalings, bias, key)
    if x.dtype != BF16:
        raise TypeError(f"bank_linear takes bfloat16 activations, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must be [..., K]")
    k = x.shape[-1]
    n, e, _ = _check_bank(k, packed, scale_bits, lora_a, lora_b, scalings, group_size, bias)
    flat = x.dim() == 2
    x2d = _aligned(x if flat else x.reshape(-1, k))
    if plan.rows != x2d.shape[0] or plan.adapters != e:
        raise ValueError(f"the plan is one of {plan.rows} rows and {plan.adapters} adapters, x has "
                         f"{x2d.shape[0]} rows and the bank {e} adapters")
    threshold = dropout_threshold(rate)
    if threshold < 65536:
        check_key(key, site, x.device)
        key = key.contiguous()
    else:
        key = None
    cfg = {"group": group_arg(group_size, k), "site": int(site), "threshold": threshold}
    frozen = (_aligned(packed), _aligned(_u16(scale_bits)),
              None if bias is None else _u16(bias).contiguous(), scalings.contiguous(), plan.buffer,
              key)
    _on_device(x2d, lora_a, lora_b, *frozen)
    grad = torch.is_grad_enabled()
    if grad and (scalings.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("scalings and bias are constants of a bank: they get no gradients")
    if grad and (x2d.requires_grad or lora_a.requires_grad or lora_b.requires_grad):
        y = BankLinearFn.apply(x2d, lora_a, lora_b, *frozen, cfg)
    else:
        a, b = lora_a, lora_b
        if a.dtype != BF16 or b.dtype != BF16:
            a, b = cast_many((a, b), BF16)
        y, _ = _forward(x2d, _aligned(a), _aligned(b), *frozen, cfg, False)
    return y if flat else y.reshape(*x.shape[:-1], n)


# ---------------------------------------------------------------------------
# the module
# ---------------------------------------------------------------------------
_ROWS: ContextVar[tuple[AdapterPlan, torch.Tensor | None] | None] = ContextVar(
    "representax_amd_adapter_rows", default=None)


@contextmanager
def adapter_rows(plan: AdapterPlan, key: torch.Tensor | None = None) -> Iterator[None]:
    """Banks called inside take each row's adapter from ``plan`` (rows in the order
    of the activations' leading axes) and their dropout from ``key``."""

    token = _ROWS.set((plan, key))
    try:
        yield
    finally:
        _ROWS.reset(token)


def active_adapter_rows() -> tuple[AdapterPlan, torch.Tensor | None] | None:
    return _ROWS.get()


class QuantizedLoRABank(torch.nn.Module):
    """One packed INT4 base projection with several adapters: the leaves of
    ``QuantizedLoRALinear`` with ``lora_a [E, r, K]`` and ``lora_b [E, N, r]``, and
    ``scalings [E]``. Called under ``adapter_rows``. ``dropout`` is the rate on the
    adapters' input while training, ``site`` the number of its masks in a step.

    It computes in bfloat16, where the linear it stands for has other arithmetic too:
    float32 activations, and float32 masters without a precision policy (which the
    linear promotes to float32), are refused, and under an fp8 policy a bank's products
    stay bfloat16."""

    def __init__(self, *, packed_weight: torch.Tensor, scale_bits: torch.Tensor,
                 bias_bits: torch.Tensor | None, lora_a: torch.Tensor, lora_b: torch.Tensor,
                 scalings: torch.Tensor, input_size: int, output_size: int,
                 group_size: int | None = None, dropout: float = 0.0, site: int = 0) -> None:
        super().__init__()
        self.input_size, self.output_size = int(input_size), int(output_size)
        self.group_size = None if group_size in (None, input_size) else int(group_size)
        n, _, _ = _check_bank(self.input_size, packed_weight, scale_bits, lora_a, lora_b, scalings,
                              self.group_size, bias_bits)
        if n != self.output_size:
            raise ValueError(f"packed weight has {n} rows, output_size is {output_size}")
        dropout_threshold(dropout)
        self.register_buffer("packed_weight", packed_weight)
        self.register_buffer("scale_bits", scale_bits)
        self.register_buffer("bias_bits", bias_bits)
        self.register_buffer("scalings", scalings)
        self.lora_a = torch.nn.Parameter(lora_a)
        self.lora_b = torch.nn.Parameter(lora_b)
        self.dropout, self.site = float(dropout), int(site)

    def _apply(self, fn, recurse: bool = True):
        """Moves with the module; a cast of its floating-point values is not for
        ``scalings``, which are no weights (an adapter has a number there)."""

        scalings = self.scalings
        super()._apply(fn, recurse)
        if self.scalings.dtype != F32:
            self.scalings = scalings.to(self.scalings.device)
        return self

    @classmethod
    def from_adapters(cls, adapters: Sequence[QuantizedLoRALinear], *, dropout: float = 0.0,
                      site: int = 0) -> "QuantizedLoRABank":
        """A bank of the adapters of one base; adapters of a smaller rank than the
        largest are extended by zeros."""

        adapters = list(adapters)
        if not adapters:
            raise ValueError("a bank needs at least one adapter")
        first = adapters[0]
        if first.packed_weight.ndim != 2:
            raise ValueError("make a bank of a stacked adapter one layer at a time (adapter[i])")
        for other in adapters[1:]:
            same = (other.group_size == first.group_size
                    and other.packed_weight.shape == first.packed_weight.shape
                    and torch.equal(other.packed_weight, first.packed_weight)
                    and torch.equal(_u16(other.scale_bits).view(torch.int16),
                                    _u16(first.scale_bits).view(torch.int16))
                    and (other.bias_bits is None) == (first.bias_bits is None)
                    and (first.bias_bits is None
                         or torch.equal(_u16(other.bias_bits).view(torch.int16),
                                        _u16(first.bias_bits).view(torch.int16))))
            if not same:
                raise ValueError("the adapters of a bank share one base weight and bias")
        rank = max(a.rank for a in adapters)
        lora_a = torch.zeros((len(adapters), rank, first.input_size), dtype=first.lora_a.dtype,
                             device=first.lora_a.device)
        lora_b = torch.zeros((len(adapters), first.output_size, rank), dtype=first.lora_b.dtype,
                             device=first.lora_b.device)
        for i, a in enumerate(adapters):
            lora_a[i, :a.rank] = a.lora_a.detach()
            lora_b[i, :, :a.rank] = a.lora_b.detach()
        scalings = torch.tensor([a.scaling for a in adapters], dtype=F32,
                                device=first.lora_a.device)
        return cls(packed_weight=first.packed_weight, scale_bits=first.scale_bits,
                   bias_bits=first.bias_bits, lora_a=lora_a, lora_b=lora_b, scalings=scalings,
                   input_size=first.input_size, output_size=first.output_size,
                   group_size=first.group_size, dropout=dropout, site=site)

    def adapter(self, index: int) -> QuantizedLoRALinear:
        """Adapter ``index`` by itself, over the same base (its rank the bank's)."""

        rank = self.lora_a.shape[1]
        return QuantizedLoRALinear(
            packed_weight=self.packed_weight, scale_bits=self.scale_bits, bias_bits=self.bias_bits,
            lora_a=self.lora_a[index].detach().clone(), lora_b=self.lora_b[index].detach().clone(),
            input_size=self.input_size, output_size=self.output_size, rank=rank,
            alpha=float(self.scalings[index]) * rank, group_size=self.group_size)

    def forward(self, value: torch.Tensor) -> torch.Tensor:
        rows = active_adapter_rows()
        if rows is None:
            raise RuntimeError("call a bank under adapter_rows(plan)")
        plan, key = rows
        value = activation_inputs(value)
        if active_compute_dtype(value.dtype) != BF16:
            raise TypeError("a bank computes in bfloat16: enter a bfloat16 precision policy")
        if compute_parameter_dtype(self.lora_a) != BF16:
            raise TypeError("float32 adapters outside a precision policy are promoted to float32, "
                            "and a bank computes in bfloat16: enter a bfloat16 precision policy, or "
                            "keep the adapters in bfloat16")
        rate = self.dropout if self.training else 0.0
        a, b = compute_operands(self.lora_a, self.lora_b)
        y = bank_linear(value.to(BF16), self.packed_weight, self.scale_bits, a, b, self.scalings,
                        plan, group_size=self.group_size, bias=self.bias_bits, rate=rate, key=key,
                        site=self.site)
        return constrain_activation(y)

    def extra_repr(self) -> str:
        e, r, _ = self.lora_a.shape
        return (f"input_size={self.input_size}, output_size={self.output_size}, adapters={e}, "
                f"rank={r}, group_size={self.group_size}, dropout={self.dropout}")


def bank_quantized_lora(models: Sequence[torch.nn.Module], *, dropout: float = 0.0):
    """One model with a bank in the place of every ``QuantizedLoRALinear``: adapter i
    of each is that of ``models[i]``. The models have one base; everything else is
    the first one's. Each bank has a ``site`` of its own. Banks compute in bfloat16
    (``QuantizedLoRABank``), and each is called by itself: the layers' fused calls
    (``gelu_mlp``, ``swiglu_mlp``, ``shared_input_projections``) are those of linears
    with one adapter."""

    models = list(models)
    if not models:
        raise ValueError("bank_quantized_lora needs at least one model")
    # a module that a model has in several places is in the list under each of them
    def places(model):
        return [n for n, m in model.named_modules(remove_duplicate=False)
                if isinstance(m, QuantizedLoRALinear)]

    paths = places(models[0])
    if not paths:
        raise ValueError("the models have no QuantizedLoRALinear modules")
    for other in models[1:]:
        if paths != places(other):
            raise ValueError("the models have their adapters in different places")
    target = copy.deepcopy(models[0])
    banks: dict[tuple[int, ...], QuantizedLoRABank] = {}
    for path in paths:
        adapters = [m.get_submodule(path) for m in models]
        key = tuple(map(id, adapters))
        if key not in banks:
            banks[key] = QuantizedLoRABank.from_adapters(adapters, dropout=dropout, site=len(banks))
            banks[key].train(target.training)
        target = _set_module(target, path, banks[key])
    return target


__all__ = ["AdapterPlan", "QuantizedLoRABank", "adapter_plan", "adapter_rows", "bank_linear",
           "bank_quantized_lora"]
