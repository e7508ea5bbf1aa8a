"""ctypes binding of ``librepresentax_amd.so`` (the C ABI in include/).

``import torch`` happens first on purpose: torch's ROCm wheel ships its own
HIP runtime under the same soname, so the library binds to that one runtime
and torch's streams and device pointers are valid inside it.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import sysconfig
from pathlib import Path

import torch  # noqa: F401  (load torch's HIP runtime before the library)

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "librepresentax_amd.so"
FAST_PATH = LIB_PATH.parent / ("_rpxfast" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

RPX_OK = 0
RPX_ERR_INVALID = 1
RPX_ERR_HIP = 2
RPX_ERR_DEVICE = 3
DTYPE_F32 = 0
DTYPE_BF16 = 1
FP8_E4M3FN = 0
FP8_E5M2 = 1
ACT_GELU = 1
ACT_SILU_MUL = 2
ACT_ADD = 3
NORM_LAYER = 0
NORM_RMS = 1
# kernel-variant knobs (rpx_set_tuning)
TUNE_INT4_TILE = 0
TUNE_BF16_TILE = 1
TUNE_FP8_TILE = 2
TUNE_SKINNY_TILE = 3
TUNE_SKINNY2 = 4
TUNE_SKINNY2_ONE = 5
TUNE_SPIN_LIMIT = 6
TUNE_GEMM_BAND = 7
TUNE_DX_PACKED = 8
TUNE_RANK_BLOCKS = 9
TUNE_RANK_NT_U = 10
TUNE_FP8_SPLITS = 11
TUNE_FP8_PAIR = 12
TUNE_MX_TILE = 13
TUNE_MX_SPLITS = 14
TUNE_MX_PAIR = 15

_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float
_size = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/representax_amd.h
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "rpx_last_error": (ctypes.c_char_p, []),
    "rpx_abi_version": (_int, []),
    "rpx_set_tuning": (_int, [_int, _int]),
    "rpx_get_tuning": (_int, [_int]),
    "rpx_check_device_errors": (_int, [_p, _p]),
    "rpx_int4_pack": (_int, [_p, _int, _i64, _i64, _i64, _p, _p, _p]),
    "rpx_int4_dequant": (_int, [_p, _p, _i64, _i64, _i64, _p, _p]),
    "rpx_int4_merge": (_int, [_p, _p, _p, _p, _i64, _i64, _i64, _i64, _f32, _p, _p]),
    "rpx_int4lora_forward_workspace": (_size, [_i64, _i64, _i64, _i64, _i64, _int]),
    "rpx_int4lora_forward": (
        _int,
        [_p, _int, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _p, _i64, _f32, _p, _p, _p, _size, _p],
    ),
    "rpx_int4lora_forward_static": (
        _int, [_p, _int, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _p, _i64, _f32, _p, _p, _p],
    ),
    "rpx_int4lora_backward_workspace": (_size, [_i64, _i64, _i64, _i64, _i64, _int]),
    "rpx_int4lora_backward": (
        _int,
        [_p, _p, _int, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _i64, _f32, _p, _p, _p, _p, _p,
         _size, _p],
    ),
    "rpx_int4lora_forward_act": (
        _int,
        [_p, _int, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _p, _i64, _f32, _int, _p, _p, _p, _p,
         _p, _size, _p],
    ),
    "rpx_int4lora_backward_act": (
        _int,
        [_p, _p, _int, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _i64, _f32, _p, _int, _p, _p, _p,
         _p, _p, _p, _p, _size, _p],
    ),
    "rpx_int4lora_forward_promoted_workspace": (_size, [_i64, _i64, _i64, _i64, _i64]),
    "rpx_int4lora_forward_promoted": (
        _int,
        [_p, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _p, _i64, _f32, _p, _p, _p, _size, _p],
    ),
    "rpx_int4lora_backward_promoted_workspace": (_size, [_i64, _i64, _i64, _i64, _i64]),
    "rpx_int4lora_backward_promoted": (
        _int,
        [_p, _p, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _i64, _f32, _p, _p, _p, _p, _p, _size,
         _p],
    ),
    "rpx_fp8_scale_workspace": (_size, [_i64]),
    "rpx_fp8_scale": (_int, [_p, _int, _i64, _int, _p, _p, _size, _p]),
    "rpx_fp8_cast": (_int, [_p, _int, _i64, _i64, _i64, _i64, _p, _int, _p, _p, _p]),
    "rpx_fp8_gemm_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_fp8_gemm": (
        _int, [_p, _int, _p, _p, _int, _p, _i64, _i64, _i64, _p, _int, _p, _size, _p]
    ),
    "rpx_fp8_linear_forward_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_fp8_linear_forward": (
        _int, [_p, _int, _i64, _i64, _p, _int, _i64, _i64, _i64, _p, _int, _p, _p, _p, _p, _size, _p]
    ),
    "rpx_fp8_linear_backward_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_fp8_linear_backward": (
        _int,
        [_p, _int, _p, _int, _i64, _i64, _i64, _i64, _i64, _p, _int, _p, _p, _p, _int, _int, _p,
         _size, _p],
    ),
    "rpx_fp8_linear_backward_codes": (
        _int, [_p, _p, _p, _i64, _i64, _i64, _p, _int, _p, _p, _int, _int, _p, _size, _p]
    ),
    "rpx_fp8_linear_backward_gemms_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_fp8_linear_backward_gemms": (
        _int, [_p, _p, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p, _int, _int, _p, _size, _p]
    ),
    "rpx_fp8_delayed_pending_words": (_size, []),
    "rpx_fp8_cast_delayed": (
        _int, [_p, _int, _i64, _i64, _i64, _i64, _int, _p, _p, _i64, _i64, _p, _p, _p]
    ),
    "rpx_fp8_cast_delayed2": (
        _int,
        [_p, _i64, _i64, _i64, _i64, _i64, _p, _p, _p, _i64, _i64, _i64, _i64, _i64, _p, _p, _int,
         _int, _p, _p, _i64, _p],
    ),
    "rpx_fp8_scale_update": (_int, [_p, _p, _p, _p, _p, _i64, _i64, _p]),
    "rpx_fp8_encode_selfcheck": (
        _int, [_int, ctypes.c_uint64, ctypes.c_uint64, _p, _p, _i64, _p]
    ),
    "rpx_host_fp8_quantize": (_int, [_p, _i64, _f32, _int, _p]),
    "rpx_int4lora_forward_multi_workspace": (_size, [_i64, _i64, _int, _p, _int]),
    "rpx_int4lora_forward_multi": (_int, [_p, _int, _i64, _i64, _int, _p, _p, _size, _p]),
    "rpx_mnr_saved_bytes": (ctypes.c_size_t, [_i64, _i64, _i64]),
    "rpx_mnr_forward": (_int, [_p, _p, _int, _i64, _i64, _i64, _f32, _p, _p, ctypes.c_size_t, _p]),
    "rpx_mnr_backward": (_int, [_p, _p, ctypes.c_size_t, _i64, _i64, _i64, _f32, _p, _p, _int, _p]),
    "rpx_cast_many": (_int, [_p, _p, _p, _i64, _p]),
    "rpx_norm_forward": (_int, [_p, _p, _p, _p, _int, _i64, _i64, _f32, _int, _p, _p, _p]),
    "rpx_norm_backward": (_int, [_p, _p, _p, _p, _int, _i64, _i64, _f32, _int, _p, _p]),
    "rpx_mxfp4_code_bytes": (_size, [_i64, _i64]),
    "rpx_mxfp4_scale_bytes": (_size, [_i64, _i64]),
    "rpx_mxfp4_quantize": (_int, [_p, _i64, _p]),
    "rpx_mxfp4_dequantize": (_int, [_p, _p, _i64, _i64, _p, _int, _p]),
    "rpx_mxfp4_gemm_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_mxfp4_gemm": (
        _int, [_p, _p, _p, _p, _i64, _i64, _i64, _p, _int, _p, _size, _p]
    ),
    "rpx_mxfp4_gated_gemm": (
        _int, [_p, _p, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p, _p, _int, _p]
    ),
    "rpx_mxfp4_gated_backward": (
        _int, [_p, _p, _p, _int, _i64, _i64, _p, _p, _p, _p, _p]
    ),
    "rpx_mxfp4_linear_saved_bytes": (_size, [_i64, _i64, _i64, _int, _int]),
    "rpx_mxfp4_linear_forward_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_mxfp4_linear_forward": (
        _int,
        [_p, _int, _i64, _i64, _i64, _p, _int, _i64, _i64, _i64, _p, _int, _p, _size, _int, _int,
         _p, _size, _p],
    ),
    "rpx_mxfp4_linear_backward_workspace": (_size, [_i64, _i64, _i64, _int, _int]),
    "rpx_mxfp4_linear_backward": (
        _int,
        [_p, _int, _i64, _i64, _i64, _p, _size, _i64, _int, _int, _p, _int, _p, _int, _p, _size,
         _p],
    ),
    "rpx_mxfp4_gated_saved_bytes": (_size, [_i64, _i64, _i64, _int, _int]),
    "rpx_mxfp4_gated_forward_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_mxfp4_gated_forward": (
        _int,
        [_p, _int, _i64, _i64, _i64, _p, _int, _i64, _i64, _p, _int, _i64, _i64, _i64, _p, _p, _p,
         _int, _p, _size, _int, _int, _p, _size, _p],
    ),
    "rpx_mxfp4_gated_backward_workspace": (_size, [_i64, _i64, _i64, _int, _int]),
    "rpx_mxfp4_gated_backward_products": (
        _int,
        [_p, _p, _p, _int, _i64, _i64, _p, _size, _i64, _int, _int, _p, _int, _p, _int, _p, _size,
         _p],
    ),
    "rpx_mxfp4_linear_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_mxfp4_linear": (
        _int, [_p, _int, _i64, _i64, _i64, _p, _p, _i64, _p, _p, _size, _p]
    ),
    "rpx_mxfp4_gated_workspace": (_size, [_i64, _i64, _i64]),
    "rpx_mxfp4_gated": (
        _int, [_p, _int, _i64, _i64, _i64, _p, _p, _p, _p, _i64, _p, _p, _size, _p]
    ),
    "rpx_adapter_plan_bytes": (_size, [_i64, _i64]),
    "rpx_adapter_plan": (_int, [_p, _int, _i64, _i64, _p, _size, _p]),
    "rpx_bank_forward_workspace": (_size, [_p, _int]),
    "rpx_bank_forward": (_int, [_p, _p, _p, _p, _size, _p]),
    "rpx_bank_backward_workspace": (_size, [_p, _int, _int, _int]),
    "rpx_bank_backward": (_int, [_p, _p, _p, _p, _p, _int, _p, _int, _p, _size, _p]),
    "rpx_dropout": (_int, [_p, _int, _i64, _p, _i64, _i64, _p, _p]),
    "rpx_block_forward": (_int, [_p, _p]),
    "rpx_block_backward_workspace": (_size, [_p, _p]),
    "rpx_block_backward": (_int, [_p, _p, _p, _size, _p]),
    "rpx_head_norm": (_int, [_p, _i64, _p, _p, _i64, _i64, _i64, _int, _p]),
}


class HeadPart(ctypes.Structure):
    """``rpx_head_part`` of include/representax_amd.h."""

    _fields_ = [(name, ctypes.c_void_p) for name in ("x", "weight", "g", "out")]
    _fields_ += [(name, ctypes.c_int64)
                 for name in ("stride_b", "stride_s", "stride_h", "heads", "repeat")]
    _fields_ += [("weight_dtype", ctypes.c_int), ("eps", ctypes.c_float)]


class BlockNorm(ctypes.Structure):
    """``rpx_block_norm`` of include/representax_amd.h."""

    _fields_ = [("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("dtype", ctypes.c_int),
                ("kind", ctypes.c_int), ("eps", ctypes.c_float)]


class Block(ctypes.Structure):
    """``rpx_block`` of include/representax_amd.h."""

    _fields_ = [("x", ctypes.c_void_p), ("u", ctypes.c_void_p), ("gate", ctypes.c_void_p),
                ("rows_per_gate", ctypes.c_int64), ("post", BlockNorm), ("norm", BlockNorm),
                ("key", ctypes.c_void_p), ("site", ctypes.c_int64), ("threshold", ctypes.c_int64),
                ("rows", ctypes.c_int64), ("size", ctypes.c_int64), ("t", ctypes.c_void_p),
                ("h", ctypes.c_void_p), ("dtype", ctypes.c_int), ("gate_dtype", ctypes.c_int),
                ("scale", ctypes.c_float)]


class BlockGradients(ctypes.Structure):
    """``rpx_block_gradients`` of include/representax_amd.h."""

    _fields_ = [(name, ctypes.c_void_p)
                for name in ("dt", "dh", "dx", "du", "d_gate", "d_weight", "d_bias",
                             "d_post_weight", "d_post_bias")]


class Bank(ctypes.Structure):
    """``rpx_bank`` of include/representax_amd.h."""

    _fields_ = [("x", ctypes.c_void_p), ("m", ctypes.c_int64), ("k", ctypes.c_int64),
                ("packed", ctypes.c_void_p), ("scale_bits", ctypes.c_void_p),
                ("n", ctypes.c_int64), ("group_size", ctypes.c_int64),
                ("bias_bits", ctypes.c_void_p), ("lora_a", ctypes.c_void_p),
                ("lora_b", ctypes.c_void_p), ("scalings", ctypes.c_void_p),
                ("adapters", ctypes.c_int64), ("rank", ctypes.c_int64), ("plan", ctypes.c_void_p),
                ("plan_bytes", ctypes.c_size_t), ("key", ctypes.c_void_p),
                ("site", ctypes.c_int64), ("threshold", ctypes.c_int64)]


class Mxfp4Part(ctypes.Structure):
    """``rpx_mxfp4_part`` of include/representax_amd.h."""

    _fields_ = [
        ("t", ctypes.c_void_p),
        ("rows", ctypes.c_int64),
        ("columns", ctypes.c_int64),
        ("row_stride", ctypes.c_int64),
        ("codes", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("code_stride", ctypes.c_int64),
        ("codes_t", ctypes.c_void_p),
        ("scales_t", ctypes.c_void_p),
        ("code_stride_t", ctypes.c_int64),
        ("dtype", ctypes.c_int),
    ]


class Int4LoraProjection(ctypes.Structure):
    """``rpx_int4lora_projection`` of include/representax_amd.h."""

    _fields_ = [
        ("packed", ctypes.c_void_p),
        ("scale_bits", ctypes.c_void_p),
        ("n", ctypes.c_int64),
        ("group_size", ctypes.c_int64),
        ("bias_bits", ctypes.c_void_p),
        ("lora_a", ctypes.c_void_p),
        ("lora_b", ctypes.c_void_p),
        ("rank", ctypes.c_int64),
        ("scaling", ctypes.c_float),
        ("y", ctypes.c_void_p),
        ("h", ctypes.c_void_p),
    ]


class NativeError(RuntimeError):
    """A HIP-side failure reported by the library."""


class DeviceError(NativeError):
    """A kernel reported a problem through the device error word."""


_LIB: ctypes.PyDLL | None = None
# These wait for the device, so other threads run meanwhile; they use no shared scratch.
_WAITING = ("rpx_check_device_errors",)


def load() -> ctypes.PyDLL:
    """Load the library, or raise: there is no fallback implementation.

    Its functions hold the interpreter's lock (as the fast-call binding's do): a call
    may enqueue several kernels over its stream's cached scratch, and no other thread's
    call may enqueue between them. None of them waits, but for ``_WAITING``."""

    global _LIB
    if _LIB is not None:
        return _LIB
    path = Path(os.environ.get("RPX_LIBRARY", LIB_PATH))
    if not path.exists():
        raise ImportError(
            f"{path} is missing; build it with `python -m representax_amd.build` "
            "(the quantized-linear path has no non-HIP implementation)"
        )
    lib, released = ctypes.PyDLL(str(path)), ctypes.CDLL(str(path))  # one loaded library
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(released if name in _WAITING else lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
        setattr(lib, name, fn)
    _LIB = lib
    return lib


_FAST = None


def fast():
    """The CPython fast-call binding of the small-M forward entry points
    (``csrc/pyfast.c``), or None where it is not built or the library was
    loaded from another path (``RPX_LIBRARY``): it links the library in its
    own directory, and a second copy of the library would not share its
    state. Callers fall back to the ctypes functions, which reach the same
    kernels."""

    global _FAST
    if _FAST is not None:
        return _FAST or None
    load()
    mod = False
    if FAST_PATH.exists() and Path(os.environ.get("RPX_LIBRARY", LIB_PATH)).resolve() == LIB_PATH:
        loader = importlib.machinery.ExtensionFileLoader("_rpxfast", str(FAST_PATH))
        spec = importlib.util.spec_from_file_location("_rpxfast", str(FAST_PATH), loader=loader)
        mod = importlib.util.module_from_spec(spec)
        loader.exec_module(mod)
    _FAST = mod
    return mod or None


def check(status: int) -> None:
    if status == RPX_OK:
        return
    msg = (load().rpx_last_error() or b"").decode(errors="replace")
    if status == RPX_ERR_INVALID:
        raise ValueError(msg)
    if status == RPX_ERR_DEVICE:
        raise DeviceError(msg)
    raise NativeError(msg)


def call(name: str, *args) -> None:
    check(getattr(load(), name)(*args))


def query(name: str, *args) -> int:
    return int(getattr(load(), name)(*args))


def block_of(fields: tuple) -> Block:
    """The fields of an ``rpx_block`` as the fast binding takes them (its norms' five in
    their places), as the structure."""

    return Block(*fields[:4], BlockNorm(*fields[4:9]), BlockNorm(*fields[9:14]), *fields[14:])


def block_forward(fields: tuple, stream) -> None:
    binding = fast()
    if binding is not None:
        check(binding.block_forward(*fields, stream))
    else:
        call("rpx_block_forward", ctypes.byref(block_of(fields)), stream)


def block_backward_workspace(fields: tuple, gradients: tuple) -> int:
    binding = fast()
    if binding is not None:
        return binding.block_backward_workspace(*fields, *gradients)
    return query("rpx_block_backward_workspace", ctypes.byref(block_of(fields)),
                 ctypes.byref(BlockGradients(*gradients)))


def block_backward(fields: tuple, gradients: tuple, workspace, nbytes: int, stream) -> None:
    binding = fast()
    if binding is not None:
        check(binding.block_backward(*fields, *gradients, workspace, nbytes, stream))
    else:
        call("rpx_block_backward", ctypes.byref(block_of(fields)),
             ctypes.byref(BlockGradients(*gradients)), workspace, nbytes, stream)


def bank_call(name: str, fields: tuple, *args) -> int:
    """``rpx_bank_<name>`` of a bank's fields: a size, or a checked status."""

    binding = fast()
    if binding is not None:
        out = getattr(binding, "bank_" + name)(*fields, *args)
    else:
        out = getattr(load(), "rpx_bank_" + name)(ctypes.byref(Bank(*fields)), *args)
    if name.endswith("_workspace"):
        return int(out)
    check(out)
    return 0
