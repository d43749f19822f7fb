"""Restatement of the 4-bit weight form in numpy, float64: w = s e q with q in -8 .. 7, e E4M3, s a float32 per matrix
(ultraquant_b200.q4; the reference has no counterpart).  Written from the definition, without the product's code."""
from __future__ import annotations

import numpy as np

# the positive finite E4M3 values by code 0 .. 126: 3 mantissa bits, exponent bias 7, subnormals of 2^-9
E4M3 = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) / 8 * 2.0 ** ((c >> 3) - 7) for c in range(127)])
# nibble (byte, half) of element i of eight
PLACE = [(0, 0), (2, 0), (0, 1), (2, 1), (1, 0), (3, 0), (1, 1), (3, 1)]


def pack(q):
    """(..., K) whole numbers -8 .. 7 -> (..., K/2) bytes."""
    u = (np.asarray(q) + 8).astype(np.uint8).reshape(*np.shape(q)[:-1], -1, 8)
    out = np.zeros((*u.shape[:-1], 4), np.uint8)
    for i, (byte, half) in enumerate(PLACE):
        out[..., byte] |= u[..., i] << (4 * half)
    return out.reshape(*u.shape[:-2], -1)


def unpack(codes):
    b = np.asarray(codes, np.uint8).reshape(*np.shape(codes)[:-1], -1, 4)
    out = np.zeros((*b.shape[:-1], 8), np.int64)
    for i, (byte, half) in enumerate(PLACE):
        out[..., i] = ((b[..., byte] >> (4 * half)) & 15).astype(np.int64) - 8
    return out.reshape(*b.shape[:-2], -1)


def e4m3_values(codes):
    """E4M3 bytes -> float64 (0x7f and 0xff: NaN)."""
    c = np.asarray(codes, np.uint8)
    mag = np.where((c & 127) == 127, np.nan, E4M3[np.minimum(c & 127, 126)])
    return np.where(c & 128, -mag, mag)


def e4m3_round(v):
    """E4M3 bytes of finite |v| <= 448: nearest, ties to the even code, +-2^-9 where v != 0 would give 0."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    lo = hi - 1
    up = (a - E4M3[lo] > E4M3[hi] - a) | ((a - E4M3[lo] == E4M3[hi] - a) & (hi % 2 == 0))
    code = np.where(up, hi, lo)
    code = np.where((code == 0) & (a != 0), 1, code)
    return (code | np.where(np.signbit(v) & (a != 0), 128, 0)).astype(np.uint8)


def matrix_scale(top, most):
    """Least power of two s >= 2^-117 with top <= most s; 1 if top is 0."""
    if top == 0:
        return np.float32(1)
    k = -117
    while top > most * 2.0 ** k:
        k += 1
    return np.float32(2.0 ** k)


def encode(W, group):
    """(N, K) -> codes, E4M3 bytes, s."""
    with np.errstate(over="ignore"):
        x = np.asarray(W).astype(np.float32).astype(np.float64)
    N, K = x.shape
    g = x.reshape(N, K // group, group)
    fine = np.isfinite(g).all(-1, keepdims=True)
    g = np.where(fine, g, 0.0)
    s = matrix_scale(np.abs(g).max() if g.size else 0.0, 3584.0)
    at = np.abs(g).argmax(-1)[..., None]        # numpy: the first of the largest
    m = np.take_along_axis(g, at, -1)[..., 0]
    e = e4m3_round(-m / (8.0 * float(s)))
    c = e4m3_values(e)[..., None] * float(s)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(c == 0, 0.0, np.clip(np.rint(g / c), -8, 7)).astype(np.int64)
    e = np.where(fine[..., 0], e, 0x7F).astype(np.uint8)
    return pack(q.reshape(N, K)), e, s


def decode(codes, e, s, group):
    return unpack(codes) * np.repeat(e4m3_values(e) * float(s), group, axis=-1)


def round_scales(c):
    """float32 group scales of one matrix -> E4M3 bytes, s."""
    c = np.asarray(c, np.float32).astype(np.float64)
    fine = np.isfinite(c)
    s = matrix_scale(np.abs(c[fine]).max() if fine.any() else 0.0, 448.0)
    return np.where(fine, e4m3_round(np.where(fine, c, 0.0) / float(s)), 0x7F).astype(np.uint8), s
