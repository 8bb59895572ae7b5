"""Block-scaled matrices and activation functions in 64 bits, from their definitions
(OCP microscaling formats MXFP4 and MXINT8; the package's counter-based random stream).

A matrix is handled line by line: `lines` is (number of lines, values of a line)."""
import math

import numpy as np

from .ref_numpy import rand_sr16

BLOCK = 32
FP4_GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
__all__ = ["ref_mx_round", "ref_mx_values", "ref_mx_pack", "ref_act", "ref_act_slope"]


def _as_lines(x, axis):
    x = np.asarray(x, dtype=np.float64)
    return x if axis == 1 else x.T


def _split(lines):
    pad = -lines.shape[1] % BLOCK
    return np.pad(lines, ((0, 0), (0, pad))).reshape(lines.shape[0], -1, BLOCK)


def ref_mx_round(x, fmt, axis=1, seed=None, stream=None):
    """what mx_quantize keeps of a matrix: (signed codes (lines, blocks, 32), scale bytes (lines, blocks),
    values shaped like x); seed and stream ask for stochastic rounding"""
    lines = _as_lines(x, axis)
    t = _split(lines)
    codes = np.zeros(t.shape, dtype=np.int64)
    scales = np.zeros(t.shape[:2], dtype=np.int64)
    values = np.zeros(t.shape)
    for i in range(t.shape[0]):
        for b in range(t.shape[1]):
            block = t[i, b]
            if not np.all(np.isfinite(block)):
                scales[i, b] = 255
                values[i, b] = np.nan
                continue
            top = np.abs(block).max()
            e = max(math.frexp(top)[1] - 1 - (2 if fmt == "fp4" else 6), -126) if top > 0 else -126
            if fmt == "fp4" and seed is not None and top > 6.0 * 2.0 ** e:
                e += 1
            a = np.abs(block) / 2.0 ** e
            if seed is not None:
                idx = np.arange(BLOCK, dtype=np.int64) + i * lines.shape[1] + b * BLOCK
                r = (rand_sr16(seed, stream, idx).astype(np.int64) >> 16) & 0xFFFF
            if fmt == "fp4" and seed is None:
                # nearest of the grid; the even code where two are as near
                dist = np.abs(a[:, None] - FP4_GRID[None, :])
                near = dist == dist.min(axis=1)[:, None]
                first = near.argmax(axis=1)
                tie = near.sum(axis=1) > 1
                q = np.where(tie & (first % 2 == 1), first + 1, first)
            elif fmt == "fp4":
                T = np.floor(a * 32768).astype(np.int64)
                bits = np.where(a < 2, 14, np.where(a < 4, 15, 16))
                q = np.minimum(((T + (r >> (16 - bits))) >> bits) + 2 * (bits - 14), 7)
            elif seed is None:
                q = np.minimum(np.rint(a), 127).astype(np.int64)
            else:
                q = np.minimum((np.floor(a * 65536).astype(np.int64) + r) >> 16, 127)
            codes[i, b] = np.where(block < 0, -q, q)
            scales[i, b] = e + 127 + (0 if fmt == "fp4" else 6)
            mag = FP4_GRID[q] if fmt == "fp4" else q.astype(np.float64)
            values[i, b] = np.where(block < 0, -mag, mag) * 2.0 ** e
    out = values.reshape(lines.shape[0], -1)[:, :lines.shape[1]]
    return codes, scales, (out if axis == 1 else out.T)


def ref_mx_pack(codes, scales, fmt):
    """the bytes of signed codes and scale bytes, as the library lays them out"""
    lines, nb = scales.shape
    if fmt == "fp4":
        nib = np.where(codes < 0, 8 - codes, codes).reshape(lines, -1)
        data = (nib[:, 0::2] | (nib[:, 1::2] << 4)).astype(np.uint8)
    else:
        data = codes.reshape(lines, -1).astype(np.int8).view(np.uint8)
    s = np.zeros((lines, -(-nb // 8) * 8), dtype=np.uint8)
    s[:, :nb] = scales
    return np.ascontiguousarray(data), s


def ref_mx_values(data, scales, fmt, shape, axis=1):
    """64-bit matrix that codes and scales of the library's layout stand for"""
    depth, lines = shape[axis], shape[1 - axis]
    nb = -(-depth // BLOCK)
    data, scales = np.asarray(data).reshape(lines, -1), np.asarray(scales).reshape(lines, -1)[:, :nb]
    if fmt == "fp4":
        nib = np.empty((lines, nb * BLOCK), dtype=np.uint8)
        nib[:, 0::2], nib[:, 1::2] = data & 15, data >> 4
        v = np.where(nib & 8, -1.0, 1.0) * FP4_GRID[nib & 7]
    else:
        v = data.view(np.int8).astype(np.float64) / 64.0
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    out = (v.reshape(lines, nb, BLOCK) * s[:, :, None]).reshape(lines, -1)[:, :depth]
    return out if axis == 1 else out.T


_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def _logistic(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def ref_act(op, z):
    z = np.asarray(z, dtype=np.float64)
    if op == "relu":
        return np.maximum(z, 0.0)
    if op == "tanh":
        return np.tanh(z)
    if op == "gelu":
        return 0.5 * z * _erfc(-z / math.sqrt(2.0))
    return _logistic(z) * (z if op == "silu" else 1.0)


def ref_act_slope(op, z):
    z = np.asarray(z, dtype=np.float64)
    if op == "relu":
        return np.where(np.isnan(z), np.nan, z > 0)
    if op == "tanh":
        return 4.0 * _logistic(2.0 * z) * _logistic(-2.0 * z)      # 1 - tanh(z)^2 without its cancellation
    if op == "gelu":
        return 0.5 * _erfc(-z / math.sqrt(2.0)) + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    s, rest = _logistic(z), _logistic(-z)
    return s * rest if op == "sig" else s * (1.0 + z * rest)
