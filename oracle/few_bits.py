"""Oracle of the operators in few bits -- TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

8-bit (e4m3) cache rows and products with 4-bit weights, in float64 from their definitions.
"""
from __future__ import annotations

import numpy as np


def _e4m3_values() -> np.ndarray:
    """The values of codes 0x00 .. 0x7e: 1 sign, 4 exponent (bias 7), 3 mantissa bits."""
    code = np.arange(127)
    exponent, mantissa = code >> 3, code & 7
    return np.where(exponent == 0, mantissa * 2.0 ** -9,
                    (1 + mantissa / 8) * 2.0 ** (exponent - 7.0))


E4M3 = _e4m3_values()


def e4m3(x) -> np.ndarray:
    """x rounded to the nearest e4m3 value, ties to the even code; |x| < 464."""
    x = np.asarray(x, dtype=np.float64)
    size = np.abs(x)
    above = np.clip(np.searchsorted(E4M3, size), 1, 126)
    low, high = E4M3[above - 1], E4M3[above]
    even_low = (above - 1) % 2 == 0
    take_low = (size - low < high - size) | ((size - low == high - size) & even_low)
    return np.copysign(np.where(take_low, low, high), x)


def coded(rows):
    """fp32 rows [..., D] as (scale fp32 [...], code values [..., D]): the scale and the quotient
    are rounded to fp32 as stated, the quotient then to e4m3."""
    rows = np.asarray(rows, dtype=np.float32)
    most = np.abs(rows).max(-1)
    finite = np.isfinite(rows).all(-1)
    least = np.maximum(most / np.float32(448), np.float32(2.0 ** -126)).astype(np.float32)
    with np.errstate(all="ignore"):
        codes = e4m3(np.where(finite[..., None], rows / least[..., None], 0).astype(np.float32))
    scale = np.where(finite, np.where(most == 0, np.float32(0), least), np.float32(np.nan))
    return scale.astype(np.float32), codes


def product(x, codes, scales, zeros, group: int):
    """x [M,K], codes [N,K], scales / zeros [G,N].  Returns x W^T and, for its tolerance,
    sum_k |x_k| s (32 + c + |z|) and sum_k |x_k| s |c - z|."""
    x, codes = np.asarray(x, np.float64), np.asarray(codes, np.float64)
    pick = np.arange(codes.shape[1]) // group
    s = np.asarray(scales, np.float64)[pick].T
    z = np.full_like(s, 8.0) if zeros is None else np.asarray(zeros, np.float64)[pick].T
    weight = (codes - z) * s
    size = np.abs(x)
    return (x @ weight.T, size @ ((32 + codes + np.abs(z)) * np.abs(s)).T,
            size @ np.abs(weight).T)
