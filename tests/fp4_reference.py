"""The FP4 operators' definitions in 64-bit numpy, for the tests: codes and scale bytes, their values, and products."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def e4m3_table() -> np.ndarray:
    """Value of every e4m3 code (finite-only: 127 and 255 are NaN)."""
    out = np.empty(256)
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        out[code] = np.nan if code & 127 == 127 else (-v if code & 128 else v)
    return out


E4M3 = e4m3_table()


def encode_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest code of non-negative values within [0, 448], ties to even."""
    values = E4M3[:127]
    hi = np.clip(np.searchsorted(values, x, side="left"), 1, 126)
    lo = hi - 1
    up = (x - values[lo] > values[hi] - x) | ((x - values[lo] == values[hi] - x) & (hi % 2 == 0))
    return np.where(up, hi, lo).astype(np.uint8)


def encode_e2m1(v: np.ndarray) -> np.ndarray:
    m = np.minimum(np.abs(v), 6.0)
    m = np.where(np.isnan(m), 0.0, m)
    hi = np.clip(np.searchsorted(GRID, m, side="left"), 1, 7)
    lo = hi - 1
    up = (m - GRID[lo] > GRID[hi] - m) | ((m - GRID[lo] == GRID[hi] - m) & (hi % 2 == 0))
    return np.where(up, hi, lo).astype(np.uint8) | (np.signbit(v).astype(np.uint8) << 3)


def mx_scale(top: np.ndarray, mode: str) -> np.ndarray:
    """e8m0 byte of a block maximum (fp32 values as float64)."""
    with np.errstate(invalid="ignore", divide="ignore"):
        target = top / 6.0 if mode == "rceil" else top
        mantissa, exponent = np.frexp(np.where(np.isfinite(target), target, 1.0))
        power = exponent - 1.0
        if mode == "rceil":
            power = power + (mantissa > 0.5)
        else:
            power = power + {"floor": 0, "ceil": mantissa > 0.5, "even": mantissa >= 0.875}[mode] - 2
        power = np.where(target == 0, -127.0, power)
        power = np.where(np.isinf(top), 127.0 if mode == "rceil" else 126.0, power)
    byte = np.clip(power, -127, 127) + 127
    return np.where(np.isnan(top), 255, byte).astype(np.uint8)


def quantize(x: np.ndarray, fmt: str, *, mode: str = "floor", second: float | None = None):
    """(codes (rows, cols), scale bytes (rows, blocks)) of a float64 matrix holding the input's exact values."""
    rows, cols = x.shape
    b = x.reshape(rows, cols // BLOCK[fmt], BLOCK[fmt])
    top = np.where(np.isnan(b).any(-1), np.nan, np.abs(np.where(np.isnan(b), 0, b)).max(-1))
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        if fmt == "mxfp4":
            byte = mx_scale(top, mode)
            unit = 2.0 ** (byte.astype(np.float64) - 127)
        else:
            s = top / 6.0
            if second is not None:
                s = (s.astype(np.float32) / np.float32(second)).astype(np.float64)
            s = np.clip(s, 0.015625, 448.0)
            byte = np.where(np.isnan(s), 127, encode_e4m3(np.where(np.isnan(s), 1.0, s))).astype(np.uint8)
            unit = np.where(byte == 127, 1.0, E4M3[byte])
            if second is not None:  # a reciprocal and a product, each rounded to fp32, as the merges do
                inverse = (np.float32(1.0) / np.float32(second)) / unit.astype(np.float32)
                return encode_e2m1(b.astype(np.float32) * inverse[..., None]).reshape(rows, cols), byte
        codes = encode_e2m1(b / unit[..., None])
    return codes.reshape(rows, cols), byte


def second_of(x: np.ndarray) -> np.float32:
    return np.float32(max(np.float32(np.abs(x).max()) / np.float32(2688.0), np.float32(2.0 ** -23)))


def values(codes: np.ndarray, byte: np.ndarray, fmt: str, second: float | None = None) -> np.ndarray:
    grid = np.concatenate([GRID, -GRID])
    unit = 2.0 ** (byte.astype(np.float64) - 127) if fmt == "mxfp4" else E4M3[byte]
    if fmt == "mxfp4":
        unit = np.where(byte == 255, np.nan, unit)
    v = grid[codes].reshape(*byte.shape, BLOCK[fmt]) * unit[..., None]
    return v.reshape(codes.shape) * (1.0 if second is None else float(second))


def unpack(packed: np.ndarray) -> np.ndarray:
    return np.stack([packed & 15, packed >> 4], axis=-1).reshape(*packed.shape[:-1], -1)


def pack(codes: np.ndarray) -> np.ndarray:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def scale_places(rows: int, blocks: int, swizzled: bool) -> np.ndarray:
    """Byte index of every scale (rows, blocks)."""
    r, c = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    if not swizzled:
        return r * blocks + c
    tiles = -(-blocks // 4)
    return ((r // 128) * tiles + c // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + c % 4


def scale_shape(rows: int, blocks: int, swizzled: bool) -> tuple[int, int]:
    return (-(-rows // 128) * 32, -(-blocks // 4) * 16) if swizzled else (rows, blocks)


def lay_out(byte: np.ndarray, swizzled: bool, padding: int = 0) -> np.ndarray:
    shape = scale_shape(*byte.shape, swizzled)
    out = np.full(shape[0] * shape[1], padding, np.uint8)
    out[scale_places(*byte.shape, swizzled)] = byte
    return out.reshape(shape)
