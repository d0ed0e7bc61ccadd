"""The INT8 products' definitions in 64 bits (numpy), and how far a result may be from them."""

from __future__ import annotations

import numpy as np

EPS = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}  # half a step
TINY = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}  # half a step of the smallest numbers


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes rint(127 x / a), ties to even, and scales a / 127 of each row. Whole-number arithmetic: every fp32 is one times
    a power of two, and 127 x, (2 m + 1) a are exact in 64 bits for numbers of 24 bits."""
    a = np.abs(x).max(axis=1, keepdims=True)
    safe = np.where(a == 0, 1.0, a)
    m = np.floor(np.abs(x) / safe * 127)
    for _ in range(2):  # the quotient may have been rounded across a whole number
        m = np.where(127 * np.abs(x) < m * safe, m - 1, np.where(127 * np.abs(x) >= (m + 1) * safe, m + 1, m))
    twice, border = 2 * 127 * np.abs(x), (2 * m + 1) * safe
    up = (twice > border) | ((twice == border) & (m % 2 == 1))
    return np.sign(x) * (m + up), a / 127


def product(x: np.ndarray, codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """(tokens, rows) for codes less their zero points (rows, cols) and scales (rows,)."""
    q, s = quantize(x)
    return (q @ codes.T) * s * scale[None, :]


def product_bound(want: np.ndarray, dtype: str) -> np.ndarray:
    """The sum is exact. fp32 roundings: of the sum, of the two products with the scales, of the token's scale and, where a
    scale is a magnitude over 127, of the row's; then that to the result's type, which for fp32 is the last of them."""
    return np.abs(want) * (5 * 2.0 ** -24 * (1 + 2.0 ** -20) + (EPS[dtype] if dtype != "float32" else 0.0)) * (1 + 2.0 ** -7) + TINY[dtype]


def gradient(dy: np.ndarray, codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    return (dy * scale[None, :]) @ codes


def gradient_bound(dy: np.ndarray, codes: np.ndarray, scale: np.ndarray, want: np.ndarray, dtype: str) -> np.ndarray:
    """Each dy * scale is rounded to fp32 (2^-24, twice where the scale is a quotient) and to 11 bits, or 22 in two terms, or
    by 2^-25 of a unit that is at most 2^-14 of the row's largest; the sum of `rows` products in fp32 on the tensor cores,
    which cut off below the last place, loses at most `rows` steps of 2^-23 a term; last the result's rounding."""
    v = np.abs(dy * scale[None, :])
    size = v @ np.abs(codes)
    terms = 2 if dtype == "float32" else 1
    off = size * (2.0 ** (-11 * terms) + 2 * 2.0 ** -24 + terms * codes.shape[0] * 2.0 ** -23)
    off += v.max(axis=1, keepdims=True) * 2.0 ** -39 * np.abs(codes).sum(axis=0)[None, :]
    return off * (1 + 2.0 ** -7) + np.abs(want) * EPS[dtype] + TINY[dtype]
