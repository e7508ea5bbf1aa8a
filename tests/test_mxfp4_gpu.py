"""MXFP4 kernels against the float64 oracle (GPU).

Bounds. Encodings and their values are exact: equal bytes. A product's float32 sum
takes one rounding per MFMA step, at most (K / 64 + 4) of them, each at most 2^-24 of
the sum of the magnitudes A = |a| |b|^T (twice that allowed for the rounding within a
step), and its output one rounding to its type: 2^-8 |S| in bf16 (8 significant bits), 2^-24 |S| in float32.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import representax_amd as rx
from oracle import mxfp4 as omx
from oracle.codecs import f32_to_bf16_bits
from representax_amd import _native as nat
from representax_amd import mxfp4, ops
from tests.helpers import DEVICE, bf16_values, from_dev, rng, to_dev, to_dev_bf16

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
POLICY = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())


def _data(g, rows, columns, scale=1.0):
    """bf16-valued rows and columns of different sizes, a zero row and a zero block."""

    t = g.standard_normal((rows, columns)) * scale
    t *= np.exp(g.standard_normal((rows, 1))) * np.exp(g.standard_normal((1, columns)))
    if rows > 4:
        t[3] = 0
    if columns > 64:
        t[:, 32:64] *= (np.arange(rows) % 2)[:, None]
    return bf16_values(t)


def _put(a, dtype):
    return to_dev_bf16(a) if dtype == BF16 else to_dev(np.asarray(a, np.float32))


def _check_product(got, a, b, dtype, what=""):
    want, size = omx.product(a, b)
    steps = a.shape[1] / 64 + 4
    bound = np.abs(want) * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24)
    bound = bound + steps * 2.0 ** -23 * size + 1e-38
    got = from_dev(got).astype(np.float64)
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), what
    off = np.abs(got - want)[~nan] - bound[~nan]
    assert off.size == 0 or off.max() <= 0, (what, off.max())


def _stored(q):
    return q.codes.cpu().numpy(), q.scales.cpu().numpy()


SHAPES = [(1, 1), (1, 32), (2, 33), (31, 31), (32, 256), (33, 257), (64, 100), (127, 512),
          (129, 130), (257, 96), (300, 777), (1, 2048), (520, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_encoding_is_the_oracles(rows, columns, dtype):
    t = _data(rng(rows * 1000 + columns), rows, columns)
    if dtype == F32:
        t = (t * 1.2345).astype(np.float32)
    along, across = rx.mxfp4_quantize_both(_put(t, dtype))
    for q, want in ((along, t), (across, t.T), (rx.mxfp4_quantize(_put(t, dtype)), t)):
        codes, scales = omx.stored(want)
        got_codes, got_scales = _stored(q)
        assert np.array_equal(got_scales, scales)
        assert np.array_equal(got_codes, codes)
        for out in (BF16, F32):
            assert np.array_equal(from_dev(q.dequantize(out)), omx.values(want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_encoding_of_extremes(dtype):
    """Largest and smallest values, subnormals, both zeros, infinities and NaN: each in
    a block of its own and in the last, partial one."""

    special = [3.38e38, -3.38e38, 2.0 ** -126, 2.0 ** -133, -0.0, np.inf, -np.inf, np.nan, 1.0,
               6.0, 7.9375, 8.0, 2.0 ** -127 * 1.5]
    t = np.zeros((len(special) * 2, 80), np.float32)
    g = rng(5)
    for i, v in enumerate(special):
        t[2 * i, 7] = v
        t[2 * i + 1] = bf16_values(g.standard_normal(80))
        t[2 * i + 1, 75] = v
    along, across = rx.mxfp4_quantize_both(_put(t, dtype))
    for q, want in ((along, t), (across, t.T)):
        codes, scales = omx.stored(want)
        got_codes, got_scales = _stored(q)
        assert np.array_equal(got_scales, scales)
        assert np.array_equal(got_codes, codes)
        values = omx.values(want)
        assert np.array_equal(from_dev(q.dequantize(F32)), values, equal_nan=True)


def test_every_bf16_value_against_every_scale():
    """All finite bf16 values next to a block's largest value of each exponent."""

    bits = np.arange(65536, dtype=np.uint32)
    v = (bits << 16).astype(np.uint32).view(np.float32)
    v = v[np.isfinite(v)]
    t = np.zeros((v.size // 16, 32), np.float32)
    t[:, :16] = v[:v.size // 16 * 16].reshape(-1, 16)
    top = np.ldexp(1.0, np.arange(t.shape[0]) % 255 - 127)
    t[:, 31] = np.maximum(top, 0)
    t = bf16_values(t)
    q = rx.mxfp4_quantize(to_dev_bf16(t))
    codes, scales = omx.stored(t)
    assert np.array_equal(_stored(q)[1], scales)
    assert np.array_equal(_stored(q)[0], codes)


def test_encoding_of_strided_and_misaligned_rows():
    g = rng(9)
    base = _data(g, 70, 400)
    for dtype in (BF16, F32):
        d = _put(base, dtype)
        for view, want in ((d[:, 3:300], base[:, 3:300]), (d[::2], base[::2]),
                           (d[5:, :256], base[5:, :256]), (d.t(), base.T),
                           (d[:, ::2], base[:, ::2]), (d[:1].expand(40, 400), base[:1].repeat(40, 0)),
                           (d.t()[7:200], base.T[7:200])):
            along, across = rx.mxfp4_quantize_both(view)
            assert np.array_equal(_stored(along)[0], omx.stored(want)[0])
            assert np.array_equal(_stored(along)[1], omx.stored(want)[1])
            assert np.array_equal(_stored(across)[0], omx.stored(want.T)[0])
            assert np.array_equal(_stored(rx.mxfp4_quantize(view))[0], omx.stored(want)[0])


PRODUCTS = [(1, 1, 1), (1, 2048, 768), (3, 17, 40), (5, 100, 2048), (16, 64, 256), (17, 300, 4096),
            (33, 130, 513), (64, 1000, 777), (65, 96, 6144), (128, 256, 256), (200, 128, 1000),
            (257, 513, 320), (300, 700, 2048), (513, 260, 96), (1, 33, 31), (1030, 520, 1500)]


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(m, n, k, out):
    g = rng(m * 7 + n * 3 + k)
    a, b = _data(g, m, k), _data(g, n, k, 0.05)
    got = rx.mxfp4_matmul(rx.mxfp4_quantize(to_dev_bf16(a)), rx.mxfp4_quantize(to_dev_bf16(b)), out)
    _check_product(got, a, b, out)


@pytest.mark.parametrize("m,n,k", [(768, 768, 8192), (96, 160, 16384), (768, 3072, 3500)])
def test_products_over_long_sums(m, n, k):
    """Few outputs and many columns, as a weight gradient has."""

    g = rng(k)
    a, b = _data(g, m, k), _data(g, n, k)
    got = rx.mxfp4_matmul(rx.mxfp4_quantize(to_dev_bf16(a)), rx.mxfp4_quantize(to_dev_bf16(b)), F32)
    _check_product(got, a, b, F32)


TILES = range(1, 6)


@pytest.mark.parametrize("tile", TILES)
def test_every_tile(tile):
    """Ragged edges, one slice to more than the pipeline holds, several bands of tiles."""

    g = rng(tile)
    for m, n, k in ((1, 1, 200), (300, 513, 256), (257, 300, 512), (513, 130, 1500),
                    (1300, 777, 700)):
        a, b = _data(g, m, k), _data(g, n, k, 0.05)
        aq, bq = rx.mxfp4_quantize(to_dev_bf16(a)), rx.mxfp4_quantize(to_dev_bf16(b))
        with ops.tuning(mx_tile=tile):
            for out in (BF16, F32):
                _check_product(rx.mxfp4_matmul(aq, bq, out), a, b, out, (tile, m, n, k))


@pytest.mark.parametrize("tile", TILES)
def test_every_tile_of_the_gated_block(tile):
    g = rng(20 + tile)
    for m, n, k in ((70, 33, 200), (300, 513, 512), (700, 260, 1500)):
        x, wg, wu = _data(g, m, k), _data(g, n, k, 0.05), _data(g, n, k, 0.05)
        xd, gd, ud = to_dev_bf16(x), to_dev_bf16(wg).requires_grad_(), to_dev_bf16(wu)
        for out in (BF16, F32):
            with ops.tuning(mx_tile=tile):
                h = mxfp4.gated_product(xd, gd.t(), ud.t(), out)
            z = h.grad_fn.saved_tensors[:2]
            _check_product(z[0], x, wg, out, "gate")
            _check_product(z[1], x, wu, out, "up")
            zg, zu = (from_dev(t).astype(np.float64) for t in z)
            want = omx.gated(zg, zu)
            bound = _silu_bound(zg, zu) + np.abs(want) * (2.0 ** -8 if out == BF16 else 2.0 ** -24)
            assert np.all(np.abs(from_dev(h.detach()) - want) <= bound)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("splits", [2, 3, 5, 64])
def test_split_sums(tile, splits):
    g = rng(tile + splits)
    m, n, k = 200, 333, 5000
    a, b = _data(g, m, k), _data(g, n, k, 0.05)
    aq, bq = rx.mxfp4_quantize(to_dev_bf16(a)), rx.mxfp4_quantize(to_dev_bf16(b))
    with ops.tuning(mx_tile=tile, mx_splits=splits):
        for out in (BF16, F32):
            _check_product(rx.mxfp4_matmul(aq, bq, out), a, b, out)


@pytest.mark.parametrize("m", [2, 40, 300])
def test_nan_blocks_reach_their_sums_only(m):
    g = rng(2)
    a, b = _data(g, m, 600), _data(g, 300, 600)
    a[1, 599] = np.nan
    b[7, 40] = np.inf
    got = rx.mxfp4_matmul(rx.mxfp4_quantize(to_dev_bf16(a)), rx.mxfp4_quantize(to_dev_bf16(b)))
    _check_product(got, a, b, BF16)
    y = rx.mxfp4_linear(to_dev_bf16(a), rx.mxfp4_quantize(to_dev_bf16(b)))
    _check_product(y, a, b, BF16)


SERVED = [(1, 6144, 2048), (1, 33, 100), (2, 2048, 6144), (4, 16, 32), (7, 1000, 777),
          (13, 2048, 6144), (16, 768, 3072), (17, 333, 512), (31, 100, 4096), (48, 129, 1030),
          (64, 768, 768), (65, 700, 300), (333, 260, 2048), (1100, 768, 256)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", SERVED)
def test_kept_weights(m, n, k, dtype):
    g = rng(m + n + k)
    x, w = _data(g, m, k), _data(g, n, k, 0.05)
    y = rx.mxfp4_linear(_put(x, dtype), rx.mxfp4_quantize(to_dev_bf16(w)))
    assert y.dtype == dtype
    _check_product(y, x, w, dtype)


@pytest.mark.parametrize("m", [1, 5, 40, 130])
def test_kept_weights_take_strided_and_misaligned_rows(m):
    g = rng(m)
    x, w = _data(g, 2 * m, 700), _data(g, 90, 515, 0.05)
    wq = rx.mxfp4_quantize(to_dev_bf16(w))
    for dtype in (BF16, F32):
        d = _put(x, dtype)
        for view, want in ((d[:m, :515], x[:m, :515]), (d[::2, 5:520], x[::2, 5:520]),
                           (d[m:, 185:], x[m:, 185:]),
                           (d[:m, :515].t().contiguous().t(), x[:m, :515])):
            _check_product(rx.mxfp4_linear(view, wq), want, w, dtype)


def _silu_bound(z_gate, z_up):
    """A bf16 or float32 output of silu(g) u evaluated in float32: the hardware
    exponential and reciprocal (a few ulps), the argument's rounding (|g| 2^-23), and
    the products; a sigmoid below float32's smallest normal number 2^-126 (g < -87) is
    zero."""

    h = omx.gated(z_gate, z_up)
    tiny = 2.0 ** -125 * (1 + np.abs(z_gate * z_up))
    return np.abs(h) * ((16 + 2 * np.abs(z_gate)) * 2.0 ** -23) + tiny


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 6144, 2048), (2, 100, 300), (13, 1300, 500),
                                   (33, 64, 257), (64, 300, 1024), (100, 520, 768),
                                   (300, 130, 512), (1001, 700, 500)])
def test_gated_block(m, n, k, dtype):
    g = rng(m * 5 + n + k)
    x, wg, wu = _data(g, m, k), _data(g, n, k, 0.05), _data(g, n, k, 0.05)
    xd = _put(x, dtype).requires_grad_()
    gd, ud = to_dev_bf16(wg).requires_grad_(), to_dev_bf16(wu).requires_grad_()
    h = mxfp4.gated_product(xd, gd.t(), ud.t(), dtype)
    z = h.grad_fn.saved_tensors[:2]
    _check_product(z[0], x, wg, dtype, "gate")
    _check_product(z[1], x, wu, dtype, "up")
    zg, zu = (from_dev(t).astype(np.float64) for t in z)
    want = omx.gated(zg, zu)
    bound = _silu_bound(zg, zu) + np.abs(want) * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24)
    assert np.all(np.abs(from_dev(h.detach()) - want) <= bound)
    with torch.no_grad():  # the same block without what a backward needs, and over kept weights
        again = mxfp4.gated_product(xd, gd.t(), ud.t(), dtype)
        kept = rx.mxfp4_gated(xd, rx.mxfp4_quantize(gd.detach()), rx.mxfp4_quantize(ud.detach()))
    near = bound + np.abs(want) * (2.0 ** -8 if dtype == BF16 else 2.0 ** -22)
    for other in (again, kept):
        # the projections are sums in another order: a rounding of theirs may differ
        _, ag = omx.product(x, wg)
        _, au = omx.product(x, wu)
        steps = (k / 64 + 4) * 2.0 ** -22
        ulp = 2.0 ** -7 if dtype == BF16 else 2.0 ** -22
        moved = (np.abs(zu) * 1.1 * (ulp * np.abs(zg) + steps * ag) + np.abs(zg) *
                 (ulp * np.abs(zu) + steps * au))
        assert np.all(np.abs(from_dev(other) - want) <= near + moved)


def _between(got, t, delta):
    """``got`` [rows, columns] decodes an encoding of some t (1 +- delta): every value
    lies among those of the two ends under the scales of the two ends."""

    lo, hi = t * (1 - delta), t * (1 + delta)
    scales = [omx.scale_bytes(v) for v in (lo, hi)]
    ends = np.stack([omx.decode(omx.encode(v, s)[0], s, t.shape[1]) for v in (lo, hi)
                     for s in scales])
    assert np.all(got >= ends.min(axis=0)) and np.all(got <= ends.max(axis=0))
    return float(np.mean(got != omx.values(t)))


def _gated_backward(dh, z, along=True, stacked=True):
    m, n = dh.shape
    wide = mxfp4._slices(n) * 256
    dz = mxfp4.MXFP4Matrix.empty(m, 2 * wide, dh.device) if along else None
    dzt = mxfp4.MXFP4Matrix.empty(2 * n, m, dh.device) if stacked else None
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    nat.call("rpx_mxfp4_gated_backward", p(dh), p(z[0]), p(z[1]), ops._dtype_code(dh.dtype), m, n,
             p(dz.codes) if along else None, p(dz.scales) if along else None,
             p(dzt.codes) if stacked else None, p(dzt.scales) if stacked else None,
             ops._stream(dh.device))
    return dz, dzt, wide


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n", [(1, 1), (5, 40), (33, 300), (64, 256), (130, 130), (257, 513),
                                 (31, 1000)])
def test_gated_backward_encodes_the_gradients(m, n, dtype):
    g = rng(m + 10 * n)
    dh, zg, zu = (_data(g, m, n, s) for s in (1e-3, 1.0, 1.0))
    dh_d, z_d = _put(dh, dtype), [_put(zg, dtype), _put(zu, dtype)]
    dz, dzt, wide = _gated_backward(dh_d, z_d)
    dg, du = omx.gated_gradients(dh.astype(np.float64), zg, zu)
    # the float32 evaluation: a few ulps and the exponential's argument
    delta = (24 + 2 * np.abs(zg).max()) * 2.0 ** -23
    got, got_t = from_dev(dz.dequantize(F32)), from_dev(dzt.dequantize(F32))
    moved = [_between(got[:, :n], dg, delta), _between(got[:, wide:wide + n], du, delta),
             _between(got_t[:n], dg.T, delta), _between(got_t[n:], du.T, delta)]
    assert max(moved) <= max(1e-3, 2.0 / (m * n))
    assert not got[:, n:wide].any() and not got[:, wide + n:].any()
    for along, stacked in ((True, False), (False, True)):
        one, one_t, _ = _gated_backward(dh_d, z_d, along, stacked)
        for a, b in ((one, dz), (one_t, dzt)):
            if a is not None:
                assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_gated_backward_of_special_values():
    """A NaN or an infinity among the inputs makes its blocks NaN and no others; a gate
    far below zero gives zero gradients."""

    m, n = 40, 96
    g = rng(4)
    dh, zg, zu = (_data(g, m, n) for _ in range(3))
    dh[3] = dh[20] = 0.25  # _data leaves row 3 zero, and parts of row 20
    zu[20] = 1.0
    dh[7, 5], zg[20, 50], zu[33, 95] = np.nan, -300.0, np.inf
    dz, dzt, wide = _gated_backward(to_dev_bf16(dh), [to_dev_bf16(zg), to_dev_bf16(zu)])
    got, got_t = from_dev(dz.dequantize(F32)), from_dev(dzt.dequantize(F32))
    for part, at in ((got[:, :n], ((7, 0), (33, 2))), (got[:, wide:wide + n], ((7, 0),))):
        want = np.zeros((m, n), bool)
        for r, b in at:
            want[r, 32 * b:32 * b + 32] = True
        assert np.array_equal(np.isnan(part), want)
    assert got[20, 50] == 0 and got[20, wide + 50] == 0
    want = np.zeros((2 * n, m), bool)
    want[5, :32], want[95, 32:], want[n + 5, :32] = True, True, True
    assert np.array_equal(np.isnan(got_t), want)


@pytest.mark.parametrize("m,k,n", [(1, 40, 24), (33, 64, 100), (100, 300, 130), (256, 768, 512),
                                   (1001, 500, 260), (3500, 768, 96), (8, 33, 1)])
def test_linear_gradients_are_the_three_products(m, k, n):
    g = rng(m + k + n)
    x, w, dy = _data(g, m, k), _data(g, n, k, 0.05), _data(g, m, n, 1e-3)
    xd, wd = to_dev_bf16(x).requires_grad_(), to_dev_bf16(w).requires_grad_()
    with rx.precision_context(POLICY):
        y = rx.linear_matmul(xd, wd.t())
    _check_product(y.detach(), x, w, BF16)
    y.backward(to_dev_bf16(dy))
    _check_product(xd.grad, dy, w.T, BF16, "dx")
    _check_product(wd.grad, dy.T, x.T, BF16, "dw")
    # a right operand that lies [K, N] gives the same codes, and one gradient alone too
    right = to_dev_bf16(w.T).requires_grad_()
    with rx.precision_context(POLICY):
        y2 = rx.linear_matmul(xd.detach(), right)
        y3 = rx.linear_matmul(xd, wd.detach().t())
    assert torch.equal(y2, y) and torch.equal(y3, y)
    assert torch.equal(torch.autograd.grad(y2, right, to_dev_bf16(dy))[0], wd.grad.t())
    assert torch.equal(torch.autograd.grad(y3, xd, to_dev_bf16(dy))[0], xd.grad)


@pytest.mark.parametrize("tile", [0, *TILES])
def test_gradients_of_one_launch_equal_two(tile):
    g = rng(30 + tile)
    for m, k, n in ((300, 520, 130), (1100, 256, 700), (64, 33, 900)):
        x, w, u = _data(g, m, k), _data(g, n, k, 0.05), _data(g, n, k, 0.05)
        dy = to_dev_bf16(_data(g, m, n, 1e-3))
        leaves = [to_dev_bf16(t).requires_grad_() for t in (x, w, u)]
        grads = []
        for pair in (-1, 0):
            with ops.tuning(mx_tile=tile, mx_pair=pair), rx.precision_context(POLICY):
                y = rx.linear_matmul(leaves[0], leaves[1].t())
                h = rx.gated_matmul(leaves[0], leaves[1].t(), leaves[2].t())
                grads.append(torch.autograd.grad(y, leaves[:2], dy) +
                             torch.autograd.grad(h, leaves, dy))
        assert all(torch.equal(a, b) for a, b in zip(*grads))
        _check_product(grads[0][1], from_dev(dy).T, x.T, BF16)


def test_linear_gradients_against_differences():
    """Operands that MXFP4 holds exactly along both axes make the product linear: moving
    one of them from 4 to 6 moves the loss by exactly the gradient times 2."""

    g = rng(11)
    pick = lambda *s: g.choice(np.array([-6, -4, -2, -1, 0, 0.5, 1, 3, 4]), s)  # noqa: E731
    m, k, n = 64, 96, 64
    x, w, dy = pick(m, k), pick(n, k), pick(m, n)
    for t in (x, w, dy):  # every block's largest magnitude within [4, 8)
        t[::32, :], t[:, ::32] = 4, 4

    def loss(xv, wv):
        with rx.precision_context(POLICY):
            y = rx.linear_matmul(xv, wv.t())
        return (y.double() * to_dev(dy)).sum(), y

    def f32(a):
        return to_dev(np.asarray(a, np.float32))

    policy_out = F32
    xd, wd = f32(x).requires_grad_(), f32(w).requires_grad_()
    y = mxfp4.linear_product(xd, wd.t(), policy_out)
    y.backward(f32(dy))
    base = float((y.detach().double() * to_dev(dy)).sum())
    for i, j in ((0, 0), (32, 17), (5, 64), (63, 32)):
        for t, other, grad, is_x in ((x, w, xd.grad, True), (w, x, wd.grad, False)):
            if t[i, j] != 4:
                continue
            moved = t.copy()
            moved[i, j] = 6
            a, b = (moved, other) if is_x else (other, moved)
            ym = mxfp4.linear_product(f32(a), f32(b).t(), policy_out)
            diff = float((ym.double() * to_dev(dy)).sum()) - base
            assert diff == 2.0 * float(grad[i, j])


@pytest.mark.parametrize("m,k,n", [(1, 40, 24), (40, 300, 130), (300, 256, 256), (1001, 500, 300)])
def test_gated_gradients_are_products_of_the_encoded_gradients(m, k, n):
    g = rng(3 * m + k + n)
    x, wg, wu = _data(g, m, k), _data(g, n, k, 0.05), _data(g, n, k, 0.05)
    dh = _data(g, m, n, 1e-3)
    xd = to_dev_bf16(x).requires_grad_()
    gd, ud = to_dev_bf16(wg).requires_grad_(), to_dev_bf16(wu).requires_grad_()
    h = mxfp4.gated_product(xd, gd.t(), ud.t(), BF16)
    z = [t.clone() for t in h.grad_fn.saved_tensors[:2]]
    h.backward(to_dev_bf16(dh))
    # the encoded gradients are checked above; here the products over them
    dz, dzt, wide = _gated_backward(to_dev_bf16(dh), z)
    dzv, dztv = (from_dev(q.dequantize(F32)).astype(np.float64) for q in (dz, dzt))

    def check(got, a, b, what):
        want, size = a @ b.T, np.abs(a) @ np.abs(b).T
        bound = np.abs(want) * 2.0 ** -8 + (a.shape[1] / 64 + 4) * 2.0 ** -23 * size + 1e-38
        assert np.all(np.abs(from_dev(got) - want) <= bound), what

    both = np.zeros((k, 2 * wide))
    both[:, :n], both[:, wide:wide + n] = omx.values(wg.T), omx.values(wu.T)
    check(xd.grad, dzv, both, "dx")
    check(gd.grad, dztv[:n], omx.values(x.T), "dgate")
    check(ud.grad, dztv[n:], omx.values(x.T), "dup")
    # any one gradient alone is the same
    for t, grad in ((xd, xd.grad), (gd, gd.grad), (ud, ud.grad)):
        leaf = t.detach().clone().requires_grad_()
        args = [leaf if t is s else s.detach() for s in (xd, gd, ud)]
        with rx.precision_context(POLICY):
            h1 = rx.gated_matmul(args[0], args[1].t(), args[2].t())
        assert torch.equal(torch.autograd.grad(h1, leaf, to_dev_bf16(dh))[0], grad)


def test_gated_gradients_against_differences():
    """The encoded gradients next to central differences of the block in float64: a
    value of a block whose scale is 2^e is at most 2^e from the one encoded (half the
    largest step) below 6 2^e and at most 2 * 2^e above."""

    m, n = 64, 64
    g = rng(8)
    dh, zg, zu = (_data(g, m, n).astype(np.float64) for _ in range(3))
    h = 1e-5
    dg = dh * (omx.gated(zg + h, zu) - omx.gated(zg - h, zu)) / (2 * h)
    du = dh * (omx.gated(zg, zu + h) - omx.gated(zg, zu - h)) / (2 * h)
    dz, _, wide = _gated_backward(to_dev_bf16(dh), [to_dev_bf16(zg), to_dev_bf16(zu)])
    got = from_dev(dz.dequantize(F32))
    for part, want in ((got[:, :n], dg), (got[:, wide:wide + n], du)):
        unit = np.repeat(2.0 ** (omx.scale_bytes(want).astype(np.float64) - 127), 32, 1)[:, :n]
        off = np.abs(part - want) / unit
        assert np.all(off <= np.where(np.abs(want) / unit > 6, 2.0, 1.0) * (1 + 1e-3) + 1e-3)


def test_broadcast_and_strided_gradients():
    g = rng(6)
    x, w = _data(g, 70, 96), _data(g, 50, 96, 0.05)
    xd, wd = to_dev_bf16(x).requires_grad_(), to_dev_bf16(w).requires_grad_()
    with rx.precision_context(POLICY):
        y = rx.linear_matmul(xd, wd.t())
        h = rx.gated_matmul(xd, wd.t(), wd.t())
    y.float().sum().backward()  # one value, expanded
    ones = np.ones((70, 50), np.float32)
    _check_product(xd.grad, ones, w.T, BF16)
    _check_product(wd.grad, ones.T, x.T, BF16)
    dy = _data(g, 50, 70)
    grads = torch.autograd.grad(h, (xd, wd), to_dev_bf16(dy).t(), retain_graph=True)
    dense = torch.autograd.grad(h, (xd, wd), to_dev_bf16(dy.T))
    assert all(torch.equal(a, b) for a, b in zip(grads, dense))  # wd is gate and up at once


def test_leading_axes_and_modules():
    g = rng(12)
    x, wg, wu, wd = (_data(g, 6 * 7, 96), _data(g, 130, 96, 0.05), _data(g, 130, 96, 0.05),
                     _data(g, 96, 130, 0.05))
    layers = [rx.Linear(_put(w, F32)) for w in (wg, wu, wd)]
    xd = to_dev_bf16(x).reshape(6, 7, 96)
    with rx.precision_context(POLICY):
        y = rx.swiglu_mlp(xd.requires_grad_(), *layers)
        y.float().square().sum().backward()
        hidden = rx.gated_matmul(xd, layers[0].weight.to(BF16).t(), layers[1].weight.to(BF16).t())
        want = rx.linear_matmul(hidden, layers[2].weight.to(BF16).t())
        kept = [rx.MXFP4Linear.from_linear(l) for l in layers]
        with torch.no_grad():
            served = rx.swiglu_mlp(xd, *kept)
            one = kept[2](hidden)
    assert y.shape == (6, 7, 96) and y.dtype == BF16
    assert torch.equal(y, want)
    assert torch.equal(one, want)
    assert xd.grad.shape == xd.shape and all(l.weight.grad.dtype == F32 for l in layers)
    assert torch.isfinite(served).all()
    scale = from_dev(want.detach()).std()
    assert np.abs(from_dev(served) - from_dev(want.detach())).max() <= 0.25 * scale
    with pytest.raises(RuntimeError, match="no gradients"):
        kept[0](xd)
    bias = rx.Linear(_put(wg, F32), torch.ones(130, device=DEVICE))
    with rx.precision_context(POLICY), torch.no_grad():
        a, b = bias(xd.detach()), rx.MXFP4Linear.from_linear(bias)(xd.detach())
    assert torch.equal(a, b)


def test_empty_operands():
    x = torch.zeros((0, 64), dtype=BF16, device=DEVICE).requires_grad_()
    w = torch.randn((48, 64), device=DEVICE).to(BF16).requires_grad_()
    with rx.precision_context(POLICY):
        y = rx.linear_matmul(x, w.t())
        h = rx.gated_matmul(x, w.t(), w.t())
    assert y.shape == h.shape == (0, 48)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert gx.shape == (0, 64) and not gw.any() and gw.shape == (48, 64)
    gx, gw = torch.autograd.grad(h, (x, w), torch.zeros_like(h))
    assert gx.shape == (0, 64) and not gw.any()
    x = torch.ones((5, 0), dtype=BF16, device=DEVICE)
    w = torch.ones((48, 0), dtype=BF16, device=DEVICE)
    wq = rx.mxfp4_quantize(w)
    assert wq.shape == (48, 0) and wq.dequantize().shape == (48, 0)
    for y in (rx.mxfp4_linear(x, wq), rx.mxfp4_gated(x, wq, wq),
              rx.mxfp4_matmul(rx.mxfp4_quantize(x), wq)):
        assert y.shape == (5, 48) and not y.any()
    none = rx.mxfp4_quantize(torch.ones((0, 64), dtype=BF16, device=DEVICE))
    assert rx.mxfp4_linear(torch.ones((5, 64), dtype=BF16, device=DEVICE), none).shape == (5, 0)


def test_another_stream_and_graph_replays():
    g = rng(13)
    w = _data(g, 300, 512, 0.05)
    wq = rx.mxfp4_quantize(to_dev_bf16(w))
    xs = [_data(g, 24, 512) for _ in range(3)]
    side = torch.cuda.Stream()
    x = to_dev_bf16(xs[0])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = rx.mxfp4_linear(x, wq)
    torch.cuda.current_stream().wait_stream(side)
    _check_product(y, xs[0], w, BF16)
    for rows in (1, 24):
        x = to_dev_bf16(xs[0][:rows])
        leaf = to_dev_bf16(w).requires_grad_()

        def step():
            with rx.precision_context(POLICY):
                out = rx.gated_matmul(x, leaf.t(), leaf.t())
                return (rx.mxfp4_linear(x, wq), rx.mxfp4_gated(x, wq, wq),
                        torch.autograd.grad(out, leaf, torch.ones_like(out))[0])

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for values in xs:
            x.copy_(to_dev_bf16(values[:rows]))
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_offsets_beyond_32_bits():
    """A matrix of more than 2^31 elements: its last rows are encoded and multiplied
    like any other's."""

    rows, columns = 1 << 20, 2304
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    t = torch.zeros((rows, columns), dtype=BF16, device=DEVICE)
    g = rng(14)
    tail = _data(g, 40, columns)
    t[-40:] = to_dev_bf16(tail)
    q = rx.mxfp4_quantize(t)
    codes, scales = omx.stored(tail)
    assert np.array_equal(q.codes[-40:].cpu().numpy(), codes)
    assert np.array_equal(q.scales[:, -40:].cpu().numpy(), scales[:, :40])
    w = _data(g, 40, columns, 0.05)
    y = rx.mxfp4_linear(t, rx.mxfp4_quantize(to_dev_bf16(w)))
    _check_product(y[-40:], tail, w, BF16)
    assert not y[:-40].any()


def test_refusals():
    x = torch.ones((4, 64), dtype=BF16, device=DEVICE)
    wq = rx.mxfp4_quantize(torch.ones((8, 64), dtype=BF16, device=DEVICE))
    other = rx.mxfp4_quantize(torch.ones((9, 64), dtype=BF16, device=DEVICE))
    with pytest.raises(ValueError, match="2-D"):
        rx.mxfp4_quantize(x[0])
    with pytest.raises(TypeError, match="dtype"):
        rx.mxfp4_quantize(x.half())
    with pytest.raises(ValueError, match="columns"):
        rx.mxfp4_linear(x[:, :32], wq)
    with pytest.raises(ValueError, match="rows"):
        rx.mxfp4_gated(x, wq, other)
    with pytest.raises(ValueError, match="product"):
        rx.mxfp4_matmul(rx.mxfp4_quantize(x[:, :32]), wq)
    with pytest.raises(TypeError, match="dtype"):
        rx.mxfp4_matmul(wq, wq, torch.float16)
    with rx.precision_context(POLICY):
        with pytest.raises(ValueError, match="right"):
            rx.linear_matmul(x, torch.ones((32, 8), dtype=BF16, device=DEVICE))
        with pytest.raises(ValueError, match="one shape"):
            rx.gated_matmul(x, torch.ones((64, 8), dtype=BF16, device=DEVICE),
                            torch.ones((64, 9), dtype=BF16, device=DEVICE))
    with pytest.raises(RuntimeError, match="ROCm"):
        rx.mxfp4_linear(x.cpu(), wq)
    with pytest.raises(ValueError, match="bias"):
        rx.MXFP4Linear(wq, torch.zeros(9, device=DEVICE))


def test_both_bindings_give_the_same_bytes(monkeypatch):
    """The CPython fast-call binding and the ctypes one reach the same kernels."""

    g = rng(77)
    m, k, n = 65, 300, 96
    x = to_dev_bf16(_data(g, m, k)).requires_grad_()
    w, u = (to_dev_bf16(_data(g, n, k, 0.1)).requires_grad_() for _ in range(2))
    dy = to_dev_bf16(_data(g, m, n))

    def everything():
        out = []
        with rx.precision_context(POLICY):
            y, h = rx.linear_matmul(x, w.t()), rx.gated_matmul(x, w.t(), u.t())
        out += [y, h, *torch.autograd.grad(y, (x, w), dy), *torch.autograd.grad(h, (x, w, u), dy)]
        q, t = rx.mxfp4_quantize_both(x.detach())
        a, b = rx.mxfp4_quantize(w.detach()), rx.mxfp4_quantize(u.detach())
        out += [q.codes, q.scales, t.codes, t.scales, t.dequantize(), a.dequantize(F32)]
        for rows in (1, 20, m):
            out += [rx.mxfp4_linear(x.detach()[:rows], a), rx.mxfp4_gated(x.detach()[:rows], a, b)]
        return out

    assert nat.fast() is not None
    fast = everything()
    monkeypatch.setattr(nat, "fast", lambda: None)
    for a, b in zip(fast, everything(), strict=True):
        assert torch.equal(a, b)


# launches of more tiles than the card holds at once: a workgroup goes from one to the next
MANY = [(1, 4100, 4099), (2, 1500, 6001)]


def _normal(seed, rows, columns, scale=1.0):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (torch.randn((rows, columns), generator=g, device=DEVICE) * scale).to(BF16)


@pytest.mark.parametrize("k", [40, 256, 300, 700, 1100])
@pytest.mark.parametrize("tile,m,n", MANY)
def test_workgroups_of_many_tiles(tile, m, n, k):
    """The bits of the small tile, whose workgroups take one each, and some rows against
    the oracle: sums of one slice, two, and more; ragged edges."""

    a, b = _normal(k, m, k), _normal(k + 1, n, k)
    aq, bq = rx.mxfp4_quantize(a), rx.mxfp4_quantize(b)
    rows = torch.tensor([0, 1, m // 2, m - 2, m - 1], device=DEVICE)
    for out in (BF16, F32):
        with ops.tuning(mx_tile=5):
            want = rx.mxfp4_matmul(aq, bq, out)
        with ops.tuning(mx_tile=tile):
            got = rx.mxfp4_matmul(aq, bq, out)
        assert torch.equal(got, want)
        _check_product(got[rows], from_dev(a[rows]), from_dev(b), out)


@pytest.mark.parametrize("k", [200, 512, 1000])
@pytest.mark.parametrize("tile,m,n", [(1, 4100, 2051), (2, 1500, 3004)])
def test_gated_workgroups_of_many_tiles(tile, m, n, k):
    x, g, u = _normal(k, m, k).requires_grad_(), _normal(k + 1, n, k), _normal(k + 2, n, k)
    for out in (BF16, F32):
        got = []
        for t in (5, tile):
            with ops.tuning(mx_tile=t):
                h = mxfp4.gated_product(x, g.t(), u.t(), out)
                with torch.no_grad():
                    got.append((h.detach(), *h.grad_fn.saved_tensors[:2],
                                mxfp4.gated_product(x, g.t(), u.t(), out)))
        assert all(torch.equal(a, b) for a, b in zip(*got, strict=True))


@pytest.mark.parametrize("tile,m,k,n", [(1, 4000, 1300, 4200), (1, 5000, 3300, 200),
                                        (2, 3000, 2100, 700), (2, 200, 5000, 3300)])
def test_two_products_of_many_tiles(tile, m, k, n):
    """Both products of a backward in one launch, sums of different lengths."""

    x, w = _normal(m, m, k).requires_grad_(), _normal(n, n, k, 0.05).requires_grad_()
    dy = _normal(k, m, n, 1e-3)
    grads = []
    for t, pair in ((5, 0), (tile, 0), (tile, -1)):
        with ops.tuning(mx_tile=t, mx_pair=pair, mx_splits=1), rx.precision_context(POLICY):
            grads.append(torch.autograd.grad(rx.linear_matmul(x, w.t()), (x, w), dy))
    for other in grads[1:]:
        assert all(torch.equal(a, b) for a, b in zip(grads[0], other, strict=True))


def test_split_sums_of_many_tiles():
    a, b = _normal(1, 2500, 5200), _normal(2, 2500, 5200, 0.05)
    aq, bq = rx.mxfp4_quantize(a), rx.mxfp4_quantize(b)
    rows = torch.tensor([0, 1300, 2499], device=DEVICE)
    with ops.tuning(mx_tile=1, mx_splits=5):
        got = rx.mxfp4_matmul(aq, bq, F32)
        with ops.tuning(mx_tile=5):
            want = rx.mxfp4_matmul(aq, bq, F32)
    assert torch.equal(got, want)
    _check_product(got[rows], from_dev(a[rows]), from_dev(b), F32)


def test_codes_beyond_32_bits():
    """More than 2^32 bytes of codes, along a matrix's rows and in the rows of its
    transpose: both encodings, a product over either axis, and the projections'
    gradients give what the last rows alone give."""

    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB of device memory")
    rows, columns, last = 1 << 22, 2304, 64
    g = rng(15)
    tail = _data(g, last, columns)
    t = torch.zeros((rows, columns), dtype=BF16, device=DEVICE)
    t[-last:] = to_dev_bf16(tail)
    along, across = rx.mxfp4_quantize_both(t)
    del t
    assert along.codes.numel() > 1 << 32 and across.codes.numel() > 1 << 32
    codes, scales = omx.stored(tail)
    assert np.array_equal(along.codes[-last:].cpu().numpy(), codes)
    assert np.array_equal(along.scales[:, -last:].cpu().numpy(), scales)
    codes, scales = omx.stored(tail.T)
    assert np.array_equal(across.codes[:, -last // 2:].cpu().numpy(), codes[:, :last // 2])
    assert np.array_equal(across.scales[-1, :, -2:].cpu().numpy(), scales[0, :, :2])
    assert not across.codes[:, :-last // 2].any() and not along.codes[:-last].any()
    w = _data(g, 40, columns, 0.05)
    y = rx.mxfp4_matmul(along, rx.mxfp4_quantize(to_dev_bf16(w)))
    _check_product(y[-last:], tail, w, BF16)
    assert not y[:-last].any()
    dy = _normal(16, 40, rows, 1e-3)
    got = rx.mxfp4_matmul(rx.mxfp4_quantize(dy), across, F32)
    _check_product(got, from_dev(dy[:, -last:]), tail.T, F32)
    del along, across, y, dy
    rows = 1 << 20
    parts = [_normal(17 + i, last, columns) for i in range(3)]
    whole = []
    for p in parts:
        whole.append(torch.zeros((rows, columns), dtype=BF16, device=DEVICE))
        whole[-1][-last:] = p
    few, few_t, _ = _gated_backward(parts[0], parts[1:])
    many, many_t, _ = _gated_backward(whole[0], whole[1:])
    assert torch.equal(many.codes[-last:], few.codes)
    assert torch.equal(many.scales[:, -last:], few.scales)
    assert torch.equal(many_t.codes[:, -last // 2:], few_t.codes[:, :last // 2])
    assert torch.equal(many_t.scales[-1, :, -2:], few_t.scales[0, :, :2])
    assert not many.codes[:-last].any()
