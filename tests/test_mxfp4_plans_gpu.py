"""Which launches MXFP4 encodings and backwards are made of (GPU)."""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd import ops
from tests.helpers import DEVICE, kernel_names

pytestmark = pytest.mark.gpu

POLICY = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())


# (11776, 768, 3072) and (16384, 3072, 768): the smaller tile, two workgroups a CU; (16384,
# 2048, 6144): a long sum of many tiles
@pytest.mark.parametrize("m,k,n,joint", [(5003, 2048, 6144, True), (4096, 2048, 2048, True),
                                         (11776, 768, 3072, True), (16384, 3072, 768, True),
                                         (16384, 2048, 6144, True), (8192, 2048, 2048, True),
                                         (16384, 768, 3072, False),
                                         (11008, 2048, 2048, False), (10240, 1024, 4096, False)])
def test_products_share_a_launch_where_the_longest_tile_ends_with_the_others(m, k, n, joint):
    g = torch.Generator(device=DEVICE).manual_seed(m + k)
    x, w, dy = (torch.randn(s, generator=g, device=DEVICE).to(torch.bfloat16)
                for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(), w.requires_grad_()
    with rx.precision_context(POLICY):
        y = rx.linear_matmul(x, w.t())
    grads, names = kernel_names(lambda: torch.autograd.grad(y, (x, w), dy, retain_graph=True))
    assert any("k_mx_gemm_pair" in name for name in names) == joint, names
    with ops.tuning(mx_pair=0):
        apart = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, apart))


# 704 and 896 waves of the form that reads once, of 800; 576 and 640, of 640
@pytest.mark.parametrize("rows,columns,dtype,once", [
    (5632, 2048, torch.bfloat16, False), (7168, 2048, torch.bfloat16, True),
    (6144, 768, torch.float32, False), (5003, 1000, torch.float32, True)])
def test_large_matrices_are_read_once_for_both_axes(rows, columns, dtype, once):
    t = torch.ones((rows, columns), device=DEVICE, dtype=dtype)
    (along, across), names = kernel_names(lambda: rx.mxfp4_quantize_both(t))
    assert any("k_mx_quantize_both" in n for n in names) == once, names
    assert any("k_mx_quantize_apart" in n for n in names) != once, names
    for q in (along, across):
        assert torch.equal(q.dequantize(dtype), torch.ones(q.shape, device=DEVICE, dtype=dtype))
