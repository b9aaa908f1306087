"""CPU restatement of the 8-bit linear path (include/kd_f8.h) in numpy:
e4m3 codes with one E8M0 scale for each 128 values, the RMS norm that writes
them and the product that reads them, in float64.

TEST INFRASTRUCTURE ONLY: results are checked against it.  Imported by tests/,
never by the product (kandinsky.cpp_amd/).

The format is the OCP one: e4m3 has a sign, 4 exponent bits (bias 7) and 3 of
mantissa, no infinities, NaN where exponent and mantissa are all ones; E8M0
byte b is 2^(b - 127), 255 NaN.
"""
from __future__ import annotations

import numpy as np

BLOCK = 128
NAN_BYTE = 255


def e4m3_values() -> np.ndarray:
    """The 256 codes' values (float64)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8.0 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


_VALUES = e4m3_values()


def round_e4m3(v: np.ndarray) -> np.ndarray:
    """Codes (uint8) of the nearest e4m3 values of |v| <= 448, ties to the
    even code; NaN as 0x7f."""
    v = np.asarray(v, dtype=np.float64)
    mag = _VALUES[:127]
    a = np.abs(np.where(np.isnan(v), 0.0, v))
    hi = np.clip(np.searchsorted(mag, a), 1, 126)
    lo = hi - 1
    dl, dh = a - mag[lo], mag[hi] - a
    c = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi))).astype(np.uint8)
    c = np.where(np.signbit(v), c | 128, c).astype(np.uint8)
    return np.where(np.isnan(v), np.uint8(0x7F), c).astype(np.uint8)


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values of uint8 codes (M, K) and scale bytes (M, blocks)."""
    s = np.where(scales == NAN_BYTE, np.nan, 2.0 ** (scales.astype(np.float64) - 127.0))
    return _VALUES[codes] * np.repeat(s, BLOCK, axis=1)[:, :codes.shape[1]]


def blocked(y: np.ndarray) -> np.ndarray:
    """(M, K) as (M, blocks, 128), zeros behind the last value."""
    M, K = y.shape
    nb = (K + BLOCK - 1) // BLOCK
    out = np.zeros((M, nb * BLOCK), dtype=np.float64)
    out[:, :K] = y
    return out.reshape(M, nb, BLOCK)


def scale_bytes(y: np.ndarray) -> np.ndarray:
    """The scale byte of each block of y (M, K): the smallest e >= -127 with
    max|y| <= 448 * 2^e, 255 where the block holds an infinity or a NaN."""
    b = blocked(y)
    bad = ~np.all(np.isfinite(b), axis=2)
    a = np.max(np.abs(np.where(np.isfinite(b), b, 0.0)), axis=2)
    table = 448.0 * 2.0 ** (np.arange(255) - 127.0)      # increasing in the byte
    return np.where(bad, NAN_BYTE, np.searchsorted(table, a, side="left")).astype(np.uint8)


def quantize(y: np.ndarray):
    """(codes uint8 (M, K), scale bytes uint8 (M, blocks))."""
    K = y.shape[1]
    s = scale_bytes(y)
    factor = np.where(s == NAN_BYTE, np.nan, 2.0 ** (127.0 - s.astype(np.float64)))
    with np.errstate(invalid="ignore"):
        v = blocked(y) * factor[:, :, None]
    return round_e4m3(v.reshape(y.shape[0], -1)[:, :K]), s


def rms_norm(s: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    """s / sqrt(mean(s^2) + eps) * weight, rows of s (float64)."""
    s = np.asarray(s, dtype=np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        return s / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)


def linear(x: np.ndarray, w: np.ndarray, bias=None) -> np.ndarray:
    """x (M, K) times w (N, K), plus bias (float64)."""
    y = x @ w.T
    return y if bias is None else y + np.asarray(bias, dtype=np.float64)
