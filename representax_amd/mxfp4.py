"""MXFP4: matrices of 4-bit floating-point numbers with one power-of-two scale
for every 32 consecutive columns of a row, products that contract the columns of
two of them, and the first half of a gated feed-forward block over them.

An extension next to the reference's INT4 weights and fp8 operands
(src/representax/models/adapters.py:38-79, src/representax/precision.py:127-221):
a third choice of matrix type, which gfx950's matrix cores multiply at twice the
rate of fp8. The format is that of the OCP Microscaling Formats specification
v1.0 (e2m1 numbers, e8m0 scales); ``include/representax_amd.h`` states it.

* ``mxfp4_quantize``, ``mxfp4_quantize_both``, ``MXFP4Matrix.dequantize``: to the
  format, along a matrix's columns or along both of its axes in one pass, and back.
* ``mxfp4_matmul``: ``a b^T`` of two encoded matrices.
* ``mxfp4_linear``, ``mxfp4_gated``: inference over kept weights, the input
  encoded within the call; ``components.MXFP4Linear`` is the module that keeps one.
* ``MXFP4LinearFn``, ``MXFP4GatedFn``: the autograd nodes that ``linear_matmul`` and
  ``gated_matmul`` take under ``PrecisionConfig.mxfp4_mixed()``. Each of a linear's
  three products has both of its operands encoded along the axis that it contracts:
  ``y = x W^T`` along the inputs, ``dx = dy W`` along the outputs, ``dW = dy^T x``
  along the tokens. The forward encodes its operands along both axes in one pass and
  keeps the codes (about half a byte per value) in place of the values.

A block that holds an infinity or a NaN stands for NaN throughout, so overflow
stays visible. Empty operands follow a product's own rules: no rows give no rows,
and a sum over nothing is zero.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .ops import BF16, F32, _aligned, _as, _dtype_code, _on_device, _ptr, _stream, _workspace

SLICE = 256  # columns are padded to this
ROW_PAD = 32  # the scales' rows are padded to this


def _slices(columns: int) -> int:
    return -(-columns // SLICE)


def _pad_rows(rows: int) -> int:
    return -(-rows // ROW_PAD) * ROW_PAD


def _scales_shape(rows: int, columns: int) -> tuple[int, int, int]:
    return (_slices(columns), _pad_rows(rows), 8)


# what ``_bytes`` is asked for: a linear's, the gated block's is one more
_SERVE, _SAVED, _FORWARD, _BACKWARD = 0, 2, 4, 6
_BYTES = ("rpx_mxfp4_linear_workspace", "rpx_mxfp4_gated_workspace",
          "rpx_mxfp4_linear_saved_bytes", "rpx_mxfp4_gated_saved_bytes",
          "rpx_mxfp4_linear_forward_workspace", "rpx_mxfp4_gated_forward_workspace",
          "rpx_mxfp4_linear_backward_workspace", "rpx_mxfp4_gated_backward_workspace")


def _bytes(what: int, m: int, n: int, k: int, need_left: bool, need_right: bool) -> int:
    """The size of a call's buffer."""

    fast = nat.fast()
    if fast is not None:
        return fast.mxfp4_bytes(what, m, n, k, need_left, need_right)
    needs = (need_left, need_right) if what in (2, 3, 6, 7) else ()
    return nat.query(_BYTES[what], m, n, k, *needs)


def _call(name: str, *args) -> None:
    """``rpx_mxfp4_<name>`` through the fast binding where it is loaded: an eager step of
    a linear is three calls whose host time would be a third ctypes' conversions."""

    fast = nat.fast()
    if fast is not None:
        nat.check(getattr(fast, "mxfp4_" + name)(*args))
    else:
        nat.call("rpx_mxfp4_" + name, *args)


class MXFP4Matrix:
    """An encoded matrix ``[rows, columns]``: ``codes`` uint8 ``[rows, C / 2]`` and
    ``scales`` uint8 ``[C / 256, R, 8]`` (C and R the columns and rows rounded up to
    256 and 32), both dense and 16-byte aligned on one device."""

    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int) -> None:
        columns = int(columns)
        cs = codes.shape
        if codes.dtype != torch.uint8 or len(cs) != 2 or cs[1] != _slices(columns) * (SLICE // 2):
            raise ValueError(f"MXFP4 codes must be uint8 [rows, {_slices(columns) * (SLICE // 2)}] "
                             f"for {columns} columns, got {codes.dtype} {tuple(cs)}")
        if scales.dtype != torch.uint8 or scales.shape != _scales_shape(cs[0], columns):
            raise ValueError(f"MXFP4 scales must be uint8 {_scales_shape(cs[0], columns)}, got "
                             f"{scales.dtype} {tuple(scales.shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("MXFP4 codes and scales must be dense")
        self.codes = codes
        self.scales = scales
        self.columns = columns

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return (self.codes.shape[0], self.columns)

    @classmethod
    def empty(cls, rows: int, columns: int, device: torch.device) -> "MXFP4Matrix":
        """Room for an encoded matrix, contents undefined."""

        made = cls.__new__(cls)  # of the right layout: without the checks
        slices = _slices(columns)
        made.codes = torch.empty((rows, slices * (SLICE // 2)), dtype=torch.uint8, device=device)
        made.scales = torch.empty((slices, _pad_rows(rows), 8), dtype=torch.uint8, device=device)
        made.columns = columns
        return made

    def dequantize(self, dtype: torch.dtype = BF16) -> torch.Tensor:
        """The values that the codes stand for (exact in bf16 and float32)."""

        codes, scales = self.codes, self.scales
        device = _on_device(codes, scales)
        rows, columns = codes.shape[0], self.columns
        out = torch.empty((rows, columns), dtype=dtype, device=device)
        with _launches_on(device):
            _call("dequantize", codes.data_ptr(), scales.data_ptr(), rows, columns,
                  out.data_ptr(), _dtype_code(dtype), _stream(device))
        return out

    def __repr__(self) -> str:
        return f"MXFP4Matrix({self.rows} x {self.columns}, {self.codes.device})"


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _launches_on(device: torch.device):
    """Context in which launches go to ``device`` (they go to the current one)."""

    if device.index is None or device.index == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(device)


def _matrix_input(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D, got shape {tuple(t.shape)}")
    if t.dtype not in (BF16, F32):
        raise TypeError(f"{what}: unsupported dtype {t.dtype}; expected float32 or bfloat16")
    return t


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    """t with its columns dense and its rows apart (any row stride)."""

    rows, columns = t.shape
    if (t.stride(1) == 1 or columns == 1) and (t.stride(0) >= columns or rows <= 1):
        return t
    return t.contiguous()


def _encode(t: torch.Tensor, along: MXFP4Matrix | None, across: MXFP4Matrix | None,
            device: torch.device) -> None:
    """``t`` (dense columns) encoded into ``along``, its transpose into ``across``."""

    rows, columns = t.shape
    outs = []
    for out in (along, across):
        outs += (None, None) if out is None else (out.codes.data_ptr(), out.scales.data_ptr())
    source = (t.data_ptr(), rows, columns, max(t.stride(0), columns))
    with _launches_on(device):
        stream = _stream(device)
        fast = nat.fast()
        if fast is not None:
            nat.check(fast.mxfp4_quantize(*source, *outs, _dtype_code(t.dtype), stream))
        else:
            part = nat.Mxfp4Part(*source, *outs[:2], 0, *outs[2:], 0, _dtype_code(t.dtype))
            nat.call("rpx_mxfp4_quantize", ctypes.byref(part), 1, stream)


def mxfp4_quantize(t: torch.Tensor) -> MXFP4Matrix:
    """``t [rows, columns]`` (bf16 or float32) encoded along its columns."""

    device = _on_device(_matrix_input(t, "MXFP4 operand"))
    if t.stride(0) == 1 and t.stride(1) > 1:  # a transpose: encode along its own rows
        base = _dense_rows(t.t())
        out = MXFP4Matrix.empty(*t.shape, device)
        _encode(base, None, out, device)
        return out
    t = _dense_rows(t)
    out = MXFP4Matrix.empty(*t.shape, device)
    _encode(t, out, None, device)
    return out


def mxfp4_quantize_both(t: torch.Tensor) -> tuple[MXFP4Matrix, MXFP4Matrix]:
    """``t`` encoded along its columns, and its transpose encoded along its own (the
    rows of ``t``), from one pass over ``t``: the operands of the two products that
    contract one axis of ``t`` each."""

    device = _on_device(_matrix_input(t, "MXFP4 operand"))
    if t.stride(0) == 1 and t.stride(1) > 1:
        across, along = mxfp4_quantize_both(t.t())
        return along, across
    t = _dense_rows(t)
    along = MXFP4Matrix.empty(*t.shape, device)
    across = MXFP4Matrix.empty(t.shape[1], t.shape[0], device)
    _encode(t, along, across, device)
    return along, across


def _gemm(a: MXFP4Matrix, b: MXFP4Matrix, out_dtype: torch.dtype, device) -> torch.Tensor:
    m, n, k = a.rows, b.rows, a.columns
    out = torch.empty((m, n), dtype=out_dtype, device=device)
    ws = _workspace(nat.query("rpx_mxfp4_gemm_workspace", m, n, k), device)
    nat.call("rpx_mxfp4_gemm", _ptr(a.codes), _ptr(a.scales), _ptr(b.codes), _ptr(b.scales), m, n,
             k, _ptr(out), _dtype_code(out_dtype), _ptr(ws), ws.numel(), _stream(device))
    return out


def _check_contraction(a: MXFP4Matrix, b: MXFP4Matrix) -> None:
    if a.columns != b.columns:
        raise ValueError(f"MXFP4 product needs a [M, K] and b [N, K]; got {a.shape} and {b.shape}")


def mxfp4_matmul(a: MXFP4Matrix, b: MXFP4Matrix, out_dtype: torch.dtype = BF16) -> torch.Tensor:
    """``a [M, K] b^T [K, N]``, summed in float32 and rounded once."""

    _check_contraction(a, b)
    device = _on_device(a.codes, a.scales, b.codes, b.scales)
    with _launches_on(device):
        return _gemm(a, b, out_dtype, device)


def _serve(x2d: torch.Tensor, weight: MXFP4Matrix, up: MXFP4Matrix | None) -> torch.Tensor:
    """``mxfp4_linear``, or ``mxfp4_gated`` with ``up``. (Written for host time, which is
    most of a single token's call: each torch attribute is read once.)"""

    _matrix_input(x2d, "x")
    if x2d.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("a product over kept MXFP4 weights gives no gradients; train a Linear "
                           "under PrecisionConfig.mxfp4_mixed(), or detach x")
    m, k = x2d.shape
    codes, scales = weight.codes, weight.scales
    n = codes.shape[0]
    if weight.columns != k or (up is not None and up.columns != k):
        raise ValueError(f"x has {k} columns, the MXFP4 weight "
                         f"{weight.columns if weight.columns != k else up.columns}")
    if up is None:
        device = _on_device(x2d, codes, scales)
    else:
        if up.codes.shape[0] != n:
            raise ValueError(f"gate and up must have the same rows, got {n} and {up.rows}")
        device = _on_device(x2d, codes, scales, up.codes, up.scales)
    x2d = _dense_rows(x2d)
    y = torch.empty((m, n), dtype=x2d.dtype, device=device)
    stream = _stream(device)
    gated = up is not None
    need = _bytes(_SERVE + gated, m, n, k, False, False)
    ws = _workspace(need, device, stream) if need else None  # none for a few rows
    args = [x2d.data_ptr(), _dtype_code(x2d.dtype), m, k, max(x2d.stride(0), k), codes.data_ptr(),
            scales.data_ptr()]
    if gated:
        args += (up.codes.data_ptr(), up.scales.data_ptr())
    with _launches_on(device):
        _call("gated" if gated else "linear", *args, n, y.data_ptr(), _ptr(ws),
              0 if ws is None else ws.numel(), stream)
    return y


def mxfp4_linear(x2d: torch.Tensor, weight: MXFP4Matrix) -> torch.Tensor:
    """``x [M, K] W^T`` in x's dtype, ``weight`` the encoded ``W [N, K]``; x is encoded
    within the call. Inference: an x that requires a gradient is refused."""

    return _serve(x2d, weight, None)


def mxfp4_gated(x2d: torch.Tensor, gate: MXFP4Matrix, up: MXFP4Matrix) -> torch.Tensor:
    """``silu(x G^T) * (x U^T)`` in x's dtype over two kept weights, in one pass over x;
    both products are rounded to x's dtype before the activation. Inference: an x that
    requires a gradient is refused."""

    return _serve(x2d, gate, up)


# ---------------------------------------------------------------------------
# autograd nodes
# ---------------------------------------------------------------------------
def _check_product(left: torch.Tensor, right: torch.Tensor, what: str) -> None:
    _matrix_input(left, f"{what}: left")
    _matrix_input(right, f"{what}: right")
    if left.shape[1] != right.shape[0]:
        raise ValueError(f"{what} needs left [M, K] and right [K, N]; got {tuple(left.shape)} "
                         f"and {tuple(right.shape)}")


def _right(t: torch.Tensor) -> torch.Tensor:
    """``t [K, N]`` as the library takes a right operand: one stride 1, the other
    spanning it (row-major, or the transposed view of a row-major weight)."""

    k, n = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 and (s0 >= n or k <= 1)) or (s0 == 1 and (s1 >= k or n <= 1)):
        return t
    return t.contiguous()


def _saved(what: int, m: int, n: int, k: int, need_left: bool, need_right: bool, device):
    """The buffer that a forward keeps for its backward, or None."""

    if not (need_left or need_right):
        return None
    return torch.empty(_bytes(what, m, n, k, need_left, need_right), dtype=torch.uint8,
                       device=device)


class MXFP4LinearFn(torch.autograd.Function):
    """``left [M, K] @ right [K, N]`` on MXFP4 operands, gradients included (see the
    module's docstring). Gradients come in the operands' dtypes."""

    @staticmethod
    def forward(ctx, left, right, out_dtype):
        _check_product(left, right, "MXFP4 linear")
        device = _on_device(left, right)
        m, k = left.shape
        n = right.shape[1]
        need_left, need_right = ctx.needs_input_grad[:2]
        x, w = _dense_rows(left), _right(right)
        y = torch.empty((m, n), dtype=out_dtype, device=device)
        saved = _saved(_SAVED, m, n, k, need_left, need_right, device)
        stream = _stream(device)
        ws = _workspace(_bytes(_FORWARD, m, n, k, False, False), device, stream)
        with _launches_on(device):
            _call("linear_forward", x.data_ptr(), _dtype_code(x.dtype), m, k,
                  x.stride(0), w.data_ptr(), _dtype_code(w.dtype), n, *w.stride(),
                  y.data_ptr(), _dtype_code(out_dtype), _ptr(saved),
                  0 if saved is None else saved.numel(), need_left, need_right, ws.data_ptr(),
                  ws.numel(), stream)
        if saved is not None:
            ctx.save_for_backward(saved)
            ctx.cfg = (m, k, n, left.dtype, right.dtype, need_left, need_right)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        m, k, n, left_dtype, right_dtype, saved_left, saved_right = ctx.cfg
        need_left, need_right = ctx.needs_input_grad[:2]
        (saved,) = ctx.saved_tensors
        device = grad.device
        g = _dense_rows(grad)
        d_left = torch.empty((m, k), dtype=left_dtype, device=device) if need_left else None
        d_right = torch.empty((n, k), dtype=right_dtype, device=device) if need_right else None
        stream = _stream(device)
        ws = _workspace(_bytes(_BACKWARD, m, n, k, need_left, need_right), device, stream)
        with _launches_on(device):
            _call("linear_backward", g.data_ptr(), _dtype_code(g.dtype), m, n,
                  g.stride(0), saved.data_ptr(), saved.numel(), k, saved_left, saved_right,
                  _ptr(d_left), _dtype_code(left_dtype), _ptr(d_right),
                  _dtype_code(right_dtype), ws.data_ptr(), ws.numel(), stream)
        return d_left, None if d_right is None else d_right.t(), None


class MXFP4GatedFn(torch.autograd.Function):
    """``silu(left @ gate) * (left @ up)``, ``left [M, K]``, ``gate`` and ``up [K, N]``:
    both projections, the activation and the product in one kernel; the backward's
    ``dx`` is one product over both projections' outputs, the two weight gradients
    another. The projections are rounded to ``out_dtype`` before the activation, as
    separate linears would leave them."""

    @staticmethod
    def forward(ctx, left, gate, up, out_dtype):
        _check_product(left, gate, "MXFP4 gated block")
        _check_product(left, up, "MXFP4 gated block")
        if gate.shape != up.shape:
            raise ValueError(f"gate and up must have one shape, got {tuple(gate.shape)} and "
                             f"{tuple(up.shape)}")
        device = _on_device(left, gate, up)
        m, k = left.shape
        n = gate.shape[1]
        need_left, need_g, need_u = ctx.needs_input_grad[:3]
        need_w = need_g or need_u
        x, wg, wu = _dense_rows(left), _right(gate), _right(up)
        h = torch.empty((m, n), dtype=out_dtype, device=device)
        z_gate = z_up = None
        if need_left or need_w:
            z_gate, z_up = (torch.empty((m, n), dtype=out_dtype, device=device) for _ in range(2))
        saved = _saved(_SAVED + 1, m, n, k, need_left, need_w, device)
        stream = _stream(device)
        ws = _workspace(_bytes(_FORWARD + 1, m, n, k, False, False), device, stream)
        with _launches_on(device):
            _call("gated_forward", x.data_ptr(), _dtype_code(x.dtype), m, k,
                  x.stride(0), wg.data_ptr(), _dtype_code(wg.dtype), *wg.stride(),
                  wu.data_ptr(), _dtype_code(wu.dtype), *wu.stride(), n, h.data_ptr(),
                  _ptr(z_gate), _ptr(z_up), _dtype_code(out_dtype), _ptr(saved),
                  0 if saved is None else saved.numel(), need_left, need_w, ws.data_ptr(),
                  ws.numel(), stream)
        if saved is not None:
            ctx.save_for_backward(z_gate, z_up, saved)
            ctx.cfg = (m, k, n, left.dtype, gate.dtype, up.dtype, need_left, need_w)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        m, k, n, left_dtype, gate_dtype, up_dtype, saved_left, saved_w = ctx.cfg
        need_left, need_g, need_u = ctx.needs_input_grad[:3]
        need_w = need_g or need_u
        z_gate, z_up, saved = ctx.saved_tensors
        device = grad.device
        dh = _aligned(_as(grad, z_gate.dtype))
        wide = gate_dtype if gate_dtype == up_dtype else F32
        d_x = torch.empty((m, k), dtype=left_dtype, device=device) if need_left else None
        d_w = torch.empty((2 * n, k), dtype=wide, device=device) if need_w else None
        stream = _stream(device)
        ws = _workspace(_bytes(_BACKWARD + 1, m, n, k, need_left, need_w), device, stream)
        with _launches_on(device):
            _call("gated_backward_products", dh.data_ptr(), z_gate.data_ptr(),
                  z_up.data_ptr(), _dtype_code(dh.dtype), m, n, saved.data_ptr(),
                  saved.numel(), k, saved_left, saved_w, _ptr(d_x), _dtype_code(left_dtype),
                  _ptr(d_w), _dtype_code(wide), ws.data_ptr(), ws.numel(), stream)
        return (d_x, _as(d_w[:n], gate_dtype).t() if need_g else None,
                _as(d_w[n:], up_dtype).t() if need_u else None, None)


def linear_product(left, right, out_dtype: torch.dtype) -> torch.Tensor:
    """``MXFP4LinearFn``, without what only a backward reads where none will run."""

    if not torch.is_grad_enabled():
        left, right = left.detach(), right.detach()
    return MXFP4LinearFn.apply(left, right, out_dtype)


def gated_product(left, gate, up, out_dtype: torch.dtype) -> torch.Tensor:
    """``MXFP4GatedFn``, without what only a backward reads where none will run."""

    if not torch.is_grad_enabled():
        left, gate, up = left.detach(), gate.detach(), up.detach()
    return MXFP4GatedFn.apply(left, gate, up, out_dtype)


__all__ = ["MXFP4GatedFn", "MXFP4LinearFn", "MXFP4Matrix", "gated_product", "linear_product",
           "mxfp4_gated", "mxfp4_linear", "mxfp4_matmul", "mxfp4_quantize", "mxfp4_quantize_both"]
