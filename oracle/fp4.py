"""4-bit floating point (mxfp4, nvfp4) restated in numpy, in 64 bits.

E2M1 codes (sign in bit 3), two per byte, the lower index in the low nibble;
mxfp4: 32 values share an E8M0 scale 2**(s - 127); nvfp4: 16 share an E4M3
scale, times one scale of the whole tensor.  Quantizing: mxfp4 takes the
largest power of two s with 4 s <= max|x| (the OCP MX rule, at least 2**-127),
nvfp4 the E4M3 value nearest to max|x| / 6; codes are the nearest E2M1 values
of x / s, ties to the even code, saturating.  A group that holds an infinity or
a NaN gets the scale's NaN code.
"""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([b / 512 if b < 8 else (1 + (b % 8) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)])
GROUP = {"mxfp4": 32, "nvfp4": 16}


def nearest(v: np.ndarray, table: np.ndarray) -> np.ndarray:
    """Index of the entry of an ascending table nearest to v >= 0, a tie to the even index."""
    mid = (table[1:] + table[:-1]) / 2
    lo, hi = np.searchsorted(mid, v, side="left"), np.searchsorted(mid, v, side="right")
    return np.where(lo == hi, lo, lo + lo % 2)


def quantize(x: np.ndarray, mode: str, global_scale: float = 1.0):
    """(codes uint8 [R, L], scale bytes uint8 [R, L / group]) of values [R, L]."""
    r, n = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = np.asarray(x, dtype=np.float64).reshape(r, -1, GROUP[mode]) / global_scale
        bad = ~np.isfinite(y).all(axis=-1)
        y = np.where(np.isfinite(y), y, 0.0)
        top = np.abs(y).max(axis=-1)
        if mode == "mxfp4":
            byte = np.clip(np.floor(np.log2(np.where(top > 0, top, 1.0))).astype(np.int64) - 2 + 127, 0, 254)
            byte = np.where(top > 0, byte, 0)
            s = 2.0 ** (byte - 127.0)
            nan = 255
        else:
            byte = nearest(top / 6, E4M3)
            s = E4M3[byte]
            nan = 127
        q = np.where(s[..., None] > 0, np.abs(y) / np.where(s > 0, s, 1.0)[..., None], 0.0)
    codes = nearest(q, E2M1) + 8 * np.signbit(y)
    return codes.reshape(r, n).astype(np.uint8), np.where(bad, nan, byte).astype(np.uint8)


def scale_values(scales: np.ndarray, mode: str) -> np.ndarray:
    b = np.asarray(scales).astype(np.int64)
    if mode == "mxfp4":
        return np.where(b == 255, np.nan, 2.0 ** (b - 127.0))
    mag = np.append(E4M3, np.nan)[b & 127]
    return np.where(b & 128, -mag, mag)


def dequantize(codes: np.ndarray, scales: np.ndarray, mode: str, global_scale: float = 1.0) -> np.ndarray:
    """The values in float64."""
    r, n = codes.shape
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return (v.reshape(r, -1, GROUP[mode]) * scale_values(scales, mode)[..., None] * global_scale).reshape(r, n)


def pack(codes: np.ndarray) -> np.ndarray:
    """[R, L] codes -> uint8 [R, L / 2]."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(b: np.ndarray) -> np.ndarray:
    out = np.empty((b.shape[0], 2 * b.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = b & 15, b >> 4
    return out


def scale_atoms(scales: np.ndarray, rows: int, K: int, mode: str) -> np.ndarray:
    """Row-major scale bytes [rows, K / group] -> the block-scaled MMA's atom
    layout (flat); bytes no row owns are 0."""
    group = GROUP[mode]
    per = 256 // group
    stages, tiles = -(-K // 256), -(-rows // 128)
    full = np.zeros((tiles * 128, stages * per), np.uint8)
    full[:rows, :K // group] = scales
    # [tile, m1, m0, stage, atom, b] -> [stage, tile, atom, m0, m1, b]
    return full.reshape(tiles, 4, 32, stages, per // 4, 4).transpose(3, 0, 4, 2, 1, 5).reshape(-1)
