"""FP8 with a scale per 128 from its definition, in 64 bits (numpy): what the block-scaled quantizers and
linear compute, without a rounding but those of their outputs."""

from __future__ import annotations

import numpy as np

from oracle.reference import e4m3_decode

BLOCK = 128
E4M3_MAX = 448.0
MIN_SCALE = 1.0 / (448.0 * 512.0)


def block_scales(y: np.ndarray, group_size: int) -> np.ndarray:
    """``max(amax / 448, 1 / (448 * 512))`` of each 128 of a row (the last may be shorter), or of the row."""
    g = group_size or y.shape[1]
    peaks = [np.abs(y[:, i:i + g]).max(axis=1) for i in range(0, y.shape[1], g)]
    return np.maximum(np.stack(peaks, axis=1) / E4M3_MAX, MIN_SCALE)


def spread(scales: np.ndarray, k: int, group_size: int) -> np.ndarray:
    """A row's scales as one value per element."""
    return np.repeat(scales, group_size or k, axis=1)[:, :k]


def half_step(v: np.ndarray) -> np.ndarray:
    """Half the distance of the e4m3 values around each |v| <= 448 (2^-9 apart below 2^-6)."""
    e = np.floor(np.log2(np.maximum(np.abs(v), 2.0**-6)))
    return np.exp2(e - 4)


def silu_mul(x: np.ndarray) -> np.ndarray:
    g, u = np.split(x.astype(np.float64), 2, axis=1)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def rmsnorm(hidden: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    h = hidden.astype(np.float64)
    return h / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps) * weight.astype(np.float64)


def linear(x8: np.ndarray, xs: np.ndarray, w8: np.ndarray, ws: np.ndarray) -> tuple[np.ndarray, ...]:
    """``(y, size, length)`` of e4m3 codes: the product, the sum of its terms' magnitudes, and the root
    of the sum of their squares."""
    n, k = w8.shape
    x = e4m3_decode(x8).astype(np.float64) * spread(xs.astype(np.float64), k, BLOCK)
    w = e4m3_decode(w8).astype(np.float64) * spread(np.repeat(ws.astype(np.float64), BLOCK, axis=0)[:n], k, BLOCK)
    return x @ w.T, np.abs(x) @ np.abs(w).T, np.sqrt((x * x) @ (w * w).T)
