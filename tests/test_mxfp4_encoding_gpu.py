"""MXFP4 encodings along both axes from one read, byte for byte against the oracle (GPU).

Large matrices take this form; each test asks the profiler that its launches did.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import representax_amd as rx
from oracle import mxfp4 as omx
from representax_amd import mxfp4
from tests.helpers import DEVICE, from_dev, kernel_names

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _matrix(seed, rows, columns, dtype):
    """Rows and columns of different sizes, zero rows and blocks, and a few values that
    make their blocks NaN, in the first rows, within, and in the last row and column."""

    g = torch.Generator(device=DEVICE).manual_seed(seed)
    t = torch.randn((rows, columns), generator=g, device=DEVICE)
    t *= torch.exp(torch.randn((rows, 1), generator=g, device=DEVICE))
    t *= torch.exp(torch.randn((1, columns), generator=g, device=DEVICE))
    t[7::97] = 0
    t[:, 32:64] *= (torch.arange(rows, device=DEVICE) % 2)[:, None]
    t[1, 5], t[rows // 2, columns // 2] = torch.nan, torch.inf
    t[rows - 1, columns - 1] = -torch.inf
    return t.to(dtype)


def _oracle(t):
    """``omx.stored`` of a large matrix, 512 rows at a time."""

    parts = [omx.stored(np.ascontiguousarray(t[i:i + 512])) for i in range(0, t.shape[0], 512)]
    return np.concatenate([c for c, _ in parts]), np.concatenate([s for _, s in parts], axis=1)


def _equal(q, want):
    codes, scales = want
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)


def _check_both(view, blocks):
    (along, across), names = kernel_names(lambda: rx.mxfp4_quantize_both(view))
    assert any("k_mx_quantize_both" in n for n in names), names
    values = from_dev(view.contiguous())
    _equal(along, _oracle(values))
    _equal(across, _oracle(values.T))
    slices = lambda n: -(-n // 256)  # noqa: E731
    rows, columns = view.shape if view.stride(1) == 1 else view.shape[::-1]
    width = 128 if view.dtype == BF16 else 64
    waves = slices(rows) * 2 * -(-slices(columns) * 256 // width)
    assert (waves // 4 <= 256) == (blocks == "few")


# launches of up to 256 workgroups are dealt to the XCDs in another order than longer ones
@pytest.mark.parametrize("dtype,rows,columns,blocks", [
    (BF16, 6001, 2051, "few"), (BF16, 7000, 3333, "many"), (F32, 5003, 1500, "few"),
    (F32, 6001, 2051, "many"), (BF16, 30011, 300, "few"), (F32, 1030, 7777, "many")])
def test_encoding_along_both_axes_from_one_read(dtype, rows, columns, blocks):
    _check_both(_matrix(rows + columns, rows, columns, dtype), blocks)


@pytest.mark.parametrize("dtype,rows,columns,blocks", [(BF16, 6001, 2051, "few"),
                                                       (F32, 5003, 1500, "few")])
def test_the_same_of_views(dtype, rows, columns, blocks):
    """Rows at odd addresses and odd distances, with values on either side of them, and a
    transposed view."""

    base = _matrix(rows, rows, columns + 9, dtype)
    _check_both(base[:, 3:3 + columns], blocks)
    _check_both(base[:, :columns].t(), blocks)


def _parts(saved, *shapes):
    """The encoded matrices that a forward keeps, in order, each part from a multiple of
    256 bytes: ``(codes, scales)`` of every shape."""

    at, out = 0, []
    for rows, columns in shapes:
        slices = -(-columns // 256)
        pair = []
        for shape in ((rows, slices * 128), (slices, -(-rows // 32) * 32, 8)):
            size = int(np.prod(shape))
            pair.append(saved[at:at + size].reshape(shape))
            at += -(-size // 256) * 256
        out.append(tuple(pair))
    assert at == saved.numel()
    return out


@pytest.mark.parametrize("right", ["weights", "operands"])  # transposed [N, K] views, or [K, N]
def test_training_codes_of_large_operands(right):
    m, k, n = 4100, 1030, 3001
    x = _matrix(1, m, k, BF16).nan_to_num(0, 0, 0)
    weights = [_matrix(2 + i, n, k, BF16).nan_to_num(0, 0, 0) for i in range(2)]
    views = [w.t() if right == "weights" else w.t().contiguous() for w in weights]
    leaves = [t.requires_grad_() for t in (x, *views)]
    h, names = kernel_names(lambda: mxfp4.gated_product(*leaves, BF16))
    assert any("k_mx_quantize_both" in name for name in names), names
    z_gate, z_up, saved = h.grad_fn.saved_tensors
    wide = -(-n // 256) * 256
    xt, both = _parts(saved, (k, m), (k, 2 * wide))
    x_host, w_host = from_dev(x.detach()), [from_dev(w) for w in weights]
    for got, want in zip(xt, _oracle(x_host.T)):
        assert np.array_equal(got.cpu().numpy(), want)
    for half, w in enumerate(w_host):
        codes, scales = _oracle(w.T)
        own = slice(half * wide // 2, (half + 1) * wide // 2)
        assert np.array_equal(both[0][:, own].cpu().numpy(), codes)
        own = slice(half * wide // 256, (half + 1) * wide // 256)
        assert np.array_equal(both[1][own].cpu().numpy(), scales)
    # the forward's own codes: a tile sums slice by slice whichever tile it is, so the
    # projections have the bits of products of separately encoded operands
    encoded = [mxfp4.MXFP4Matrix(*(torch.from_numpy(t).to(DEVICE) for t in _oracle(v)), k)
               for v in (x_host, *w_host)]
    assert torch.equal(z_gate, rx.mxfp4_matmul(encoded[0], encoded[1]))
    assert torch.equal(z_up, rx.mxfp4_matmul(encoded[0], encoded[2]))


def test_training_codes_of_operands_of_two_types():
    """A bf16 input with a float32 master: two launches, one for each type."""

    m, k, n = 4100, 1030, 3001
    x = _matrix(5, m, k, BF16).nan_to_num(0, 0, 0).requires_grad_()
    w = _matrix(6, n, k, F32).nan_to_num(0, 0, 0).requires_grad_()
    y, names = kernel_names(lambda: mxfp4.linear_product(x, w.t(), F32))
    assert sum("k_mx_quantize_both" in name for name in names) == 2, names
    (saved,) = y.grad_fn.saved_tensors
    xt, wt = _parts(saved, (k, m), (k, n))
    for got, t in ((xt, x), (wt, w)):
        for a, b in zip(got, _oracle(from_dev(t.detach()).T)):
            assert np.array_equal(a.cpu().numpy(), b)
    encoded = [mxfp4.MXFP4Matrix(*(torch.from_numpy(v).to(DEVICE)
                                   for v in _oracle(from_dev(t.detach()))), k) for t in (x, w)]
    assert torch.equal(y, rx.mxfp4_matmul(*encoded, F32))
