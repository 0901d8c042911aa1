"""64-bit restatement of the operators on 8-bit floating-point blocks (test infrastructure only).

Written from the definitions: e4m3 codes by their bits, the smallest power of two that brings a
block's largest finite magnitude to 448 or below, codes rounded to nearest even, every sum in float64.
"""
from __future__ import annotations

import math

import numpy as np

BLOCK = 128


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def _code_value(c: int) -> float:
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    if (c & 127) == 127:
        return math.nan
    v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
    return -v if s else v


VALUES = np.array([_code_value(c) for c in range(256)])  # float64 value of every code
_POSITIVE = VALUES[:127]                                 # ascending


def encode(v: np.ndarray) -> np.ndarray:
    """Codes of float64 values of magnitude <= 448, nearest, ties to the even code; NaN to 0x7f."""
    v = np.asarray(v, dtype=np.float64)
    a = np.abs(np.where(np.isnan(v), 0.0, v))
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _POSITIVE[lo], _POSITIVE[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(np.signbit(v), c | 128, c)
    return np.where(np.isnan(v), 127, c).astype(np.uint8)


def spread(scale: np.ndarray, rows: int, shape) -> np.ndarray:
    """A scale per value, float64: scale [ceil(R/rows), ceil(C/128)] over shape (R, C)."""
    s = np.repeat(np.repeat(scale.astype(np.float64), rows, 0), BLOCK, 1)
    return s[:shape[0], :shape[1]]


def scale_of(top: float) -> float:
    if not top > 0:
        return 1.0
    e = math.frexp(top / 448)[1] - 2
    while 448 * 2.0 ** e < top:
        e += 1
    return 2.0 ** max(e, -126)


def quantize(x: np.ndarray, rows: int = 1):
    """(codes uint8, scale float32) of x [M, K], any float dtype."""
    x = np.asarray(x, dtype=np.float64)
    M, K = x.shape
    finite = np.isfinite(x)
    a = np.where(finite, np.abs(x), 0.0)
    scale = np.ones((-(-M // rows), blocks(K)), np.float32)
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            scale[i, j] = scale_of(a[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK].max(initial=0.0))
    with np.errstate(invalid="ignore"):
        return encode(np.where(finite, x / spread(scale, rows, x.shape), math.nan)), scale


def values(codes: np.ndarray, scale: np.ndarray, rows: int = 1) -> np.ndarray:
    return VALUES[codes] * spread(scale, rows, codes.shape)


def act(v: np.ndarray, kind: int) -> np.ndarray:
    """ActivationType by its number: none, exact GELU, ReLU, SiLU, HardSwish, tanh."""
    if kind == 1:
        return v * np.vectorize(lambda t: 0.5 * math.erfc(-t / math.sqrt(2)), otypes=[float])(v)
    if kind == 2:
        return np.where(v < 0, 0.0, v)
    if kind == 3:
        return v / (1 + np.exp(-v))
    if kind == 4:
        return v * np.clip(v / 6 + 0.5, 0, 1)
    return np.tanh(v) if kind == 5 else v


def slope(v: np.ndarray, kind: int) -> np.ndarray:
    if kind == 1:
        cdf = np.vectorize(lambda t: 0.5 * math.erfc(-t / math.sqrt(2)), otypes=[float])(v)
        return cdf + v * np.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if kind == 2:
        return (v > 0).astype(np.float64)
    if kind == 3:
        s = 1 / (1 + np.exp(-v))
        return s + v * s * (1 - s)
    if kind == 4:
        return np.where(v <= -3, 0.0, np.where(v >= 3, 1.0, v / 3 + 0.5))
    return 1 / np.cosh(v) ** 2 if kind == 5 else np.ones_like(v)
