"""MXFP4 in numpy and float64: blocks of 32 values with one power-of-two scale and
4-bit e2m1 codes (OCP Microscaling Formats specification v1.0), the products of such
matrices and the gated feed-forward block over them. No reference counterpart."""

from __future__ import annotations

import numpy as np

BLOCK = 32
SLICE = 256
ROW_PAD = 32
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NAN_SCALE = 255


def _blocks(t: np.ndarray) -> np.ndarray:
    rows, columns = t.shape
    count = -(-columns // BLOCK)
    out = np.zeros((rows, count * BLOCK))
    out[:, :columns] = t
    return out.reshape(rows, count, BLOCK)


def scale_bytes(t: np.ndarray) -> np.ndarray:
    """``uint8 [rows, blocks]``: e + 127, or 255 for a block that is not finite."""

    v = np.abs(_blocks(np.asarray(t, np.float64)))
    bad = ~np.isfinite(v).all(axis=-1)
    top = np.where(np.isfinite(v), v, 0.0).max(axis=-1)
    _, exponent = np.frexp(np.where(top > 0, top, 1.0))
    e = np.where(top > 0, np.maximum(exponent - 1 - 2, -127), -127)
    return np.where(bad, NAN_SCALE, e + 127).astype(np.uint8)


def nearest_code(a: np.ndarray) -> np.ndarray:
    """Codes 0..7 of magnitudes: the nearest level, ties to the even code."""

    a = np.asarray(a, np.float64)
    d = np.abs(a[..., None] - LEVELS)
    first = d.argmin(axis=-1)  # the lower of two equally near levels
    second = np.minimum(first + 1, 7)
    tie = np.take_along_axis(d, first[..., None], -1)[..., 0] == \
        np.take_along_axis(d, second[..., None], -1)[..., 0]
    return np.where(tie & (first % 2 == 1), second, first).astype(np.uint8)


def encode(t: np.ndarray, scales: np.ndarray | None = None):
    """``(codes uint8 [rows, blocks * 32], scale bytes [rows, blocks])``."""

    v = _blocks(np.asarray(t, np.float64))
    s = scale_bytes(t) if scales is None else scales
    finite = s != NAN_SCALE
    a = np.where(finite[..., None], np.where(np.isfinite(v), v, 0.0), 0.0)
    a = np.ldexp(a, 127 - s.astype(np.int32)[..., None])
    code = nearest_code(np.abs(a)) | (np.signbit(a).astype(np.uint8) << 3)
    return code.reshape(v.shape[0], -1), s


def decode(code: np.ndarray, scales: np.ndarray, columns: int) -> np.ndarray:
    """float64 ``[rows, columns]``."""

    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = v.reshape(code.shape[0], -1, BLOCK)
    s = scales.astype(np.int32)[..., None]
    out = np.where(s == NAN_SCALE, np.nan, np.ldexp(v, s - 127))
    return out.reshape(code.shape[0], -1)[:, :columns]


def values(t: np.ndarray) -> np.ndarray:
    """What the encoding of ``t`` along its columns stands for."""

    t = np.asarray(t)
    return decode(*encode(t), t.shape[1])


def stored(t: np.ndarray):
    """``(codes, scales)`` as the library lays them out."""

    rows, columns = t.shape
    code, s = encode(t)
    slices = -(-columns // SLICE)
    wide = np.zeros((rows, slices * SLICE), np.uint8)
    wide[:, :code.shape[1]] = code
    scales = np.zeros((-(-rows // ROW_PAD) * ROW_PAD, slices * 8), np.uint8)
    scales[:rows, :s.shape[1]] = s
    scales = scales.reshape(-1, slices, 8).transpose(1, 0, 2)
    return wide[:, 0::2] | (wide[:, 1::2] << 4), np.ascontiguousarray(scales)


def product(a: np.ndarray, b: np.ndarray):
    """``(A B^T, |A| |B|^T)`` of the encodings of a [M, K] and b [N, K]."""

    av, bv = values(a), values(b)
    with np.errstate(invalid="ignore"):
        return av @ bv.T, np.abs(av) @ np.abs(bv).T


def sigmoid(g: np.ndarray) -> np.ndarray:
    e = np.exp(-np.abs(g))
    return np.where(g >= 0, 1.0, e) / (1.0 + e)


def gated(z_gate: np.ndarray, z_up: np.ndarray) -> np.ndarray:
    return z_gate * sigmoid(z_gate) * z_up


def gated_gradients(dh: np.ndarray, z_gate: np.ndarray, z_up: np.ndarray):
    """``(dz_gate, dz_up)`` of ``gated``."""

    s = sigmoid(z_gate)
    return dh * z_up * s * (1.0 + z_gate * sigmoid(-z_gate)), dh * z_gate * s


__all__ = ["decode", "encode", "gated", "gated_gradients", "nearest_code", "product",
           "scale_bytes", "sigmoid", "stored", "values"]
