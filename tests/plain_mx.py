"""Microscaling formats, plainly: float64 numpy on the CPU, a value at a time in its meaning and a table for the numbers."""

import math

import numpy as np

GROUP = 32
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3_table():
    out = []
    for byte in range(127):  # (127 is NaN)
        e, m = byte >> 3, byte & 7
        out.append(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return np.array(out)


E4M3 = _e4m3_table()


def scale_byte(amax, emax):
    """The byte of a group whose largest magnitude is amax; 255 for one that is no number."""
    if not math.isfinite(amax):
        return 255
    if amax == 0:
        return 0
    m, x = math.frexp(amax)  # amax = m 2^x, m in [1/2, 1)
    return max(x - 1 - emax + (2 * m > 1.75) + 127, 0)


def nearest(v, table):
    """The index of the number nearest to |v|, ties to the even index; past the last number, the last."""
    v = np.abs(v)
    hi = np.clip(np.searchsorted(table, v), 0, len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = v - table[lo], table[hi] - v
    pick_hi = (above < below) | ((above == below) & (hi % 2 == 0))
    return np.where(pick_hi | (v >= table[-1]), hi, lo)


def quantize(y, table, emax):
    """float64 rows [n, d] -> (codes with the sign in the bit above the index's, bytes [n, groups])."""
    n, d = y.shape
    groups = -(-d // GROUP)
    g = np.zeros((n, groups * GROUP))
    g[:, :d] = y
    g = g.reshape(n, groups, GROUP)
    with np.errstate(invalid="ignore"):
        amax = np.where(np.isfinite(g).all(axis=2), np.abs(g).max(axis=2), np.inf)
    s = np.array([[scale_byte(a, emax) for a in row] for row in amax]).reshape(n, groups)
    v = np.where((s == 255)[:, :, None], 0.0, g) * 2.0 ** (127 - np.where(s == 255, 127, s))[:, :, None]
    sign = np.where((s == 255)[:, :, None], 0, np.signbit(v))
    bit = 8 if len(table) == 8 else 128
    return (nearest(v, table) + sign * bit).reshape(n, -1)[:, :d].astype(np.uint8), s.astype(np.uint8)


def values(codes, scales, table):
    """What codes [n, d] and bytes [n, groups] stand for, float64; NaN in groups of byte 255."""
    bit = 8 if len(table) == 8 else 128
    idx = codes & (bit - 1)
    v = np.where(idx < len(table), table[np.minimum(idx, len(table) - 1)], np.nan) * np.where(codes & bit, -1.0, 1.0)
    p = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.int64) - 127))
    return v * np.repeat(p, GROUP, axis=1)[:, : codes.shape[1]]


def two_a_byte(codes):
    """4-bit codes [n, d] as bytes [n, ceil(d / 2)], the first in the low half."""
    n, d = codes.shape
    c = np.zeros((n, d + d % 2), dtype=np.uint8)
    c[:, :d] = codes
    return c[:, 0::2] | (c[:, 1::2] << 4)


def gelu(v, kind):
    if kind == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if kind == "gelu_erf":
        return 0.5 * v * (1 + np.vectorize(math.erf)(v / math.sqrt(2)))
    return v / (1 + np.exp(-v)) if kind == "silu" else v
