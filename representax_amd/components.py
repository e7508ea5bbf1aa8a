"""The native projection that the adapter replaces
(mirror of src/representax/models/components.py:58-94), and its form with a kept
4-bit weight for inference."""

from __future__ import annotations

import torch

from .mxfp4 import MXFP4Matrix, mxfp4_linear, mxfp4_quantize
from .precision import activation_inputs, compute_parameter, linear_matmul


def _generator(key) -> torch.Generator | None:
    if key is None or isinstance(key, torch.Generator):
        return key
    g = torch.Generator()
    g.manual_seed(int(key))
    return g


class Linear(torch.nn.Module):
    """Batched linear projection ``y = x W^T (+ b)`` with ``W [*, N, K]``.

    ``__call__`` follows components.py:81-94: inputs are cast to the activation
    dtype, the fp32 master weight to the compute dtype, and the product goes
    through ``linear_matmul`` (so the fp8 policy reaches the fp8 kernels).
    """

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        self.weight = torch.nn.Parameter(weight)
        self.bias = None if bias is None else torch.nn.Parameter(bias)

    @classmethod
    def init(cls, input_size: int, output_size: int, *, key, scale: float,
             dtype: torch.dtype = torch.float32, bias: bool = False,
             device: torch.device | str | None = None) -> "Linear":
        """``weight = scale * N(0, 1)`` of shape ``[output, input]``, zero bias
        (components.py:65-79). ``key`` is an int seed or a torch.Generator."""

        w = scale * torch.randn((output_size, input_size), generator=_generator(key), dtype=dtype)
        b = torch.zeros((output_size,), dtype=dtype) if bias else None
        if device is not None:
            w = w.to(device)
            b = None if b is None else b.to(device)
        return cls(w, b)

    @property
    def input_size(self) -> int:
        return self.weight.shape[-1]

    @property
    def output_size(self) -> int:
        return self.weight.shape[-2]

    def forward(self, value: torch.Tensor) -> torch.Tensor:
        value = activation_inputs(value)
        weight = compute_parameter(self.weight)
        output = linear_matmul(value, weight.transpose(-1, -2), fp8_owner=self)
        if self.bias is not None:
            output = output + compute_parameter(self.bias)
        return output


class MXFP4Linear(torch.nn.Module):
    """A frozen projection ``y = x W^T (+ b)`` whose weight is kept in MXFP4 (0.53 bytes
    a value), for inference (an extension): the input is cast to the activation dtype
    and encoded within the call, so the result is that of a ``Linear`` under
    ``PrecisionConfig.mxfp4_mixed()`` without encoding the weight on every call."""

    def __init__(self, weight: MXFP4Matrix, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        if bias is not None and tuple(bias.shape) != (weight.rows,):
            raise ValueError(f"bias: shape {tuple(bias.shape)}, expected {(weight.rows,)}")
        self.input_size = weight.columns
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, linear: Linear) -> "MXFP4Linear":
        """Encodes the compute view of a native ``Linear``'s weight ``[N, K]``."""

        weight = compute_parameter(linear.weight.detach())
        bias = None if linear.bias is None else linear.bias.detach().clone()
        return cls(mxfp4_quantize(weight), bias)

    @property
    def output_size(self) -> int:
        return self.codes.shape[0]

    @property
    def weight(self) -> MXFP4Matrix:
        return MXFP4Matrix(self.codes, self.scales, self.input_size)

    def inputs(self, value: torch.Tensor) -> torch.Tensor:
        """``value`` as rows in the activation dtype."""

        return activation_inputs(value).reshape(-1, self.input_size)

    def forward(self, value: torch.Tensor) -> torch.Tensor:
        y = mxfp4_linear(self.inputs(value), self.weight)
        if self.bias is not None:
            y = y + compute_parameter(self.bias).to(y.dtype)
        return y.reshape(*value.shape[:-1], self.output_size)


__all__ = ["Linear", "MXFP4Linear"]
