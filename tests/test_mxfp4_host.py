"""MXFP4 host logic: layout, policy and refusals (CPU only, nothing launched)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import representax_amd as rx
from oracle import mxfp4 as omx
from representax_amd import _native as nat

P = 16  # a pointer that is never dereferenced: validation fails first
BF16 = nat.DTYPE_BF16


@pytest.mark.parametrize("rows,columns", [(1, 1), (32, 256), (33, 257), (768, 3072), (6144, 2048)])
def test_sizes_match_the_layout(rows, columns):
    codes, scales = omx.stored(torch.zeros((rows, columns)).numpy())
    assert nat.query("rpx_mxfp4_code_bytes", rows, columns) == codes.size
    assert nat.query("rpx_mxfp4_scale_bytes", rows, columns) == scales.size
    m = rx.MXFP4Matrix(torch.from_numpy(codes), torch.from_numpy(scales), columns)
    assert m.shape == (rows, columns) and m.rows == rows


def test_sizes_of_nothing():
    for rows, columns in ((0, 5), (5, 0), (-1, 5)):
        assert nat.query("rpx_mxfp4_code_bytes", rows, columns) == 0
        assert nat.query("rpx_mxfp4_scale_bytes", rows, columns) == 0
        assert nat.query("rpx_mxfp4_linear_workspace", rows, 8, columns) == 0


def test_matrix_refuses_other_layouts():
    codes, scales = (torch.from_numpy(t) for t in omx.stored(torch.ones((40, 300)).numpy()))
    with pytest.raises(ValueError, match="codes"):
        rx.MXFP4Matrix(codes[:, :128], scales, 300)
    with pytest.raises(ValueError, match="codes"):
        rx.MXFP4Matrix(codes.view(torch.int8), scales, 300)
    with pytest.raises(ValueError, match="scales"):
        rx.MXFP4Matrix(codes, scales[:1], 300)
    with pytest.raises(ValueError, match="codes"):
        rx.MXFP4Matrix(codes, scales, 600)
    with pytest.raises(ValueError, match="dense"):
        rx.MXFP4Matrix(codes.t().contiguous().t(), scales, 300)


def test_policy():
    cfg = rx.PrecisionConfig.mxfp4_mixed()
    assert (cfg.compute_dtype, cfg.resolved_matrix_dtype) == ("bfloat16", "float4_e2m1fn")
    policy = rx.resolve_precision_policy(cfg)
    assert policy.matrix_dtype == torch.float4_e2m1fn_x2
    assert rx.PrecisionConfig.model_validate(cfg.model_dump()) == cfg


def test_cpu_tensors_fail_loudly():
    policy = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())
    x, w = torch.ones((4, 64), dtype=torch.bfloat16), torch.ones((8, 64), dtype=torch.bfloat16)
    with rx.precision_context(policy):
        with pytest.raises(RuntimeError, match="ROCm"):
            rx.linear_matmul(x, w.t())
        with pytest.raises(RuntimeError, match="ROCm"):
            rx.gated_matmul(x, w.t(), w.t())
    with pytest.raises(RuntimeError, match="ROCm"):
        rx.mxfp4_quantize(x)


def test_gated_matmul_without_the_policy_is_separate_products():
    x, g, u = torch.randn(3, 4, 8), torch.randn(8, 6), torch.randn(8, 6)
    want = torch.nn.functional.silu(x @ g) * (x @ u)
    torch.testing.assert_close(rx.gated_matmul(x, g, u), want)
    layers = [rx.Linear(t) for t in (g.t(), u.t(), torch.randn(8, 6))]
    torch.testing.assert_close(rx.swiglu_mlp(x, *layers), want @ layers[2].weight.t())


def test_c_entries_refuse_before_any_launch():
    def part(**over):
        fields = dict(t=P, rows=4, columns=8, row_stride=8, codes=P, scales=P, code_stride=0,
                      codes_t=None, scales_t=None, code_stride_t=0, dtype=BF16)
        fields.update(over)
        return (nat.Mxfp4Part * 1)(nat.Mxfp4Part(**fields))

    for over, match in ((dict(dtype=7), "dtype"), (dict(rows=-1), "extents"),
                        (dict(scales=None), "together"), (dict(codes=None, scales=None), "output"),
                        (dict(t=None), "null"), (dict(row_stride=7), "overlap"),
                        (dict(code_stride=64), "stride"), (dict(code_stride=136), "stride"),
                        (dict(codes=8), "aligned"),
                        (dict(codes_t=P, scales_t=8), "aligned"),
                        (dict(columns=1 << 40, row_stride=1 << 40), "extents")):
        with pytest.raises(ValueError, match=match):
            nat.call("rpx_mxfp4_quantize", part(**over), 1, None)
    with pytest.raises(ValueError, match="count"):
        nat.call("rpx_mxfp4_quantize", part(), 5, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_quantize", None, 1, None)
    with pytest.raises(ValueError, match="dtype"):
        nat.call("rpx_mxfp4_dequantize", P, P, 4, 8, P, 9, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_dequantize", P, None, 4, 8, P, BF16, None)
    with pytest.raises(ValueError, match="extents"):
        nat.call("rpx_mxfp4_gemm", P, P, P, P, -1, 8, 8, P, BF16, None, 0, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_gemm", P, P, P, None, 8, 8, 8, P, BF16, None, 0, None)
    with pytest.raises(ValueError, match="aligned"):
        nat.call("rpx_mxfp4_gemm", P, 8, P, P, 8, 8, 8, P, BF16, None, 0, None)
    with pytest.raises(ValueError, match="together"):
        nat.call("rpx_mxfp4_gated_gemm", P, P, P, P, P, P, 8, 8, 8, P, P, None, BF16, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_gated_gemm", P, P, P, P, None, P, 8, 8, 8, P, None, None, BF16, None)
    with pytest.raises(ValueError, match="output"):
        nat.call("rpx_mxfp4_gated_backward", P, P, P, BF16, 8, 8, None, None, None, None, None)
    with pytest.raises(ValueError, match="together"):
        nat.call("rpx_mxfp4_gated_backward", P, P, P, BF16, 8, 8, P, None, None, None, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_linear", None, BF16, 4, 64, 64, P, P, 8, P, P, 1 << 20, None)
    with pytest.raises(ValueError, match="overlap"):
        nat.call("rpx_mxfp4_linear", P, BF16, 4, 64, 63, P, P, 8, P, P, 1 << 20, None)
    m, n, k = 4096, 768, 768  # takes a workspace whatever kernel serves it
    need = nat.query("rpx_mxfp4_linear_workspace", m, n, k)
    assert need >= m * k // 2
    with pytest.raises(ValueError, match="workspace too small"):
        nat.call("rpx_mxfp4_linear", P, BF16, m, k, k, P, P, n, P, P, need - 1, None)
    need = nat.query("rpx_mxfp4_gated_workspace", m, n, k)
    with pytest.raises(ValueError, match="workspace too small"):
        nat.call("rpx_mxfp4_gated", P, BF16, m, k, k, P, P, P, P, n, P, P, need - 1, None)
    assert ctypes.sizeof(nat.Mxfp4Part) == 88


def test_training_entries_refuse_before_any_launch():
    big = 1 << 30

    def forward(left=P, right=P, y=P, left_stride=64, strides=(1, 64), saved=P, saved_bytes=big,
                ws=P, ws_bytes=big, dtype=BF16):
        nat.call("rpx_mxfp4_linear_forward", left, dtype, 40, 64, left_stride, right, BF16, 48,
                 *strides, y, BF16, saved, saved_bytes, 1, 1, ws, ws_bytes, None)

    need = nat.query("rpx_mxfp4_linear_saved_bytes", 40, 48, 64, 1, 1)
    assert need > nat.query("rpx_mxfp4_linear_saved_bytes", 40, 48, 64, 1, 0) > 0
    assert nat.query("rpx_mxfp4_linear_saved_bytes", 40, 48, 64, 0, 0) == 0
    for over, match in ((dict(dtype=5), "dtype"), (dict(left=None), "null"), (dict(y=None), "null"),
                        (dict(left_stride=63), "overlap"), (dict(strides=(2, 64)), "stride"),
                        (dict(strides=(1, 63)), "stride"), (dict(right=None), "null"),
                        (dict(saved=None), "saved buffer"), (dict(saved_bytes=need - 1), "saved"),
                        (dict(saved=8), "aligned"), (dict(ws_bytes=100), "workspace too small"),
                        (dict(ws=None), "workspace too small")):
        with pytest.raises(ValueError, match=match):
            forward(**over)

    def backward(grad=P, saved=P, saved_bytes=big, d_left=P, d_right=P, need=(1, 1), ws_bytes=big):
        nat.call("rpx_mxfp4_linear_backward", grad, BF16, 40, 48, 48, saved, saved_bytes, 64, *need,
                 d_left, BF16, d_right, BF16, P, ws_bytes, None)

    for over, match in ((dict(grad=None), "null"), (dict(need=(0, 1)), "saved nothing"),
                        (dict(saved_bytes=need - 1), "saved"), (dict(d_left=8), "aligned"),
                        (dict(ws_bytes=100), "workspace too small")):
        with pytest.raises(ValueError, match=match):
            backward(**over)
    backward(d_left=None, d_right=None)  # nothing asked for

    def gated(z_gate=P, z_up=P, saved_bytes=big, ws_bytes=big, up=P):
        nat.call("rpx_mxfp4_gated_forward", P, BF16, 40, 64, 64, P, BF16, 1, 64, up, BF16, 1, 64,
                 48, P, z_gate, z_up, BF16, P, saved_bytes, 1, 1, P, ws_bytes, None)

    need = nat.query("rpx_mxfp4_gated_saved_bytes", 40, 48, 64, 1, 1)
    for over, match in ((dict(z_up=None), "together"), (dict(z_gate=8), "aligned"),
                        (dict(saved_bytes=need - 1), "saved"), (dict(up=None), "null"),
                        (dict(ws_bytes=100), "workspace too small")):
        with pytest.raises(ValueError, match=match):
            gated(**over)
    with pytest.raises(ValueError, match="saved nothing"):
        nat.call("rpx_mxfp4_gated_backward_products", P, P, P, BF16, 40, 48, P, big, 64, 1, 0, P,
                 BF16, P, BF16, P, big, None)
    with pytest.raises(ValueError, match="null"):
        nat.call("rpx_mxfp4_gated_backward_products", None, P, P, BF16, 40, 48, P, big, 64, 1, 1, P,
                 BF16, P, BF16, P, big, None)


@pytest.mark.parametrize("shape", [(1, 2048, 6144), (13, 6144, 2048), (65, 300, 777),
                                   (768, 768, 16384), (1001, 500, 1300), (0, 64, 64), (64, 0, 64)])
def test_fast_binding_sizes_and_validates_as_the_library_does(shape):
    fast, lib = nat.fast(), nat.load()
    assert fast is not None
    for what, name in enumerate(rx.mxfp4._BYTES):
        for left in (False, True):
            for right in (False, True):
                needs = (int(left), int(right)) if what in (2, 3, 6, 7) else ()
                assert fast.mxfp4_bytes(what, *shape, left, right) == getattr(lib, name)(*shape, *needs)
    with pytest.raises(ValueError):
        fast.mxfp4_bytes(len(rx.mxfp4._BYTES), *shape, 1, 1)


def test_fast_binding_refuses():
    fast = nat.fast()
    p = 16  # never dereferenced: validation fails first
    with pytest.raises(ValueError, match="overlap"):
        nat.check(fast.mxfp4_quantize(p, 4, 64, 32, p, p, None, None, nat.DTYPE_BF16, None))
    with pytest.raises(ValueError, match="no output"):
        nat.check(fast.mxfp4_quantize(p, 4, 64, 64, None, None, None, None, nat.DTYPE_BF16, None))
    with pytest.raises(ValueError, match="aligned"):
        nat.check(fast.mxfp4_quantize(p, 4, 64, 64, 8, p, None, None, nat.DTYPE_BF16, None))
    with pytest.raises(ValueError, match="null"):
        nat.check(fast.mxfp4_dequantize(None, p, 4, 64, p, nat.DTYPE_BF16, None))
    with pytest.raises(ValueError, match="workspace"):
        nat.check(fast.mxfp4_linear(p, nat.DTYPE_BF16, 65, 64, 64, p, p, 64, p, None, 0, None))
    for name in ("quantize", "dequantize", "linear", "gated", "linear_forward", "linear_backward",
                 "gated_forward", "gated_backward_products"):
        with pytest.raises(TypeError):
            getattr(fast, "mxfp4_" + name)(p)
