"""The paged key-value cache and its attention from their definitions, in 64 bits (numpy), token by token."""

from __future__ import annotations

import numpy as np


def rotate(x: np.ndarray, cos_sin: np.ndarray, positions: np.ndarray, interleaved: bool) -> np.ndarray:
    """``x [T, heads, d]``: each pair of the first ``rot`` elements as a complex number times e^(i angle)."""
    rot = cos_sin.shape[1]
    first = np.arange(rot // 2) * 2 if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    out = x.astype(np.float64).copy()
    for t, p in enumerate(positions):
        turn = cos_sin[p, :rot // 2].astype(np.float64) + 1j * cos_sin[p, rot // 2:].astype(np.float64)
        z = (out[t][:, first] + 1j * out[t][:, second]) * turn
        out[t][:, first], out[t][:, second] = z.real, z.imag
    return out


def tokens(cache: np.ndarray, scale: np.ndarray | None, table: np.ndarray, begin: int, end: int) -> np.ndarray:
    """Tokens ``[begin, end)`` of a sequence ``[n, heads, d]``, those of a page that is not there left out."""
    pages, _, page, _ = cache.shape
    i = np.arange(begin, end)
    at = table[i // page].astype(np.int64)
    there = (at >= 0) & (at < pages)
    at, off = at[there], i[there] % page
    x = cache[at, :, off].astype(np.float64)
    return x if scale is None else x * scale[at, :, off].astype(np.float64)[..., None]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> tuple[np.ndarray, ...]:
    """``(out, size, spread)`` of ``q [q_heads, d]`` over ``k``, ``v [n, heads, d]``: the attention, the same sum of
    the values' magnitudes, and each head's largest sum of the magnitudes of a score's products."""
    heads, group = k.shape[1], q.shape[0] // k.shape[1]
    out, size, spread = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[0])
    if k.shape[0] == 0:
        return out, size, spread
    for j in range(q.shape[0]):
        kj, vj = k[:, j // group], v[:, j // group]
        s = kj @ q[j] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[j], size[j] = p @ vj, p @ np.abs(vj)
        spread[j] = (np.abs(kj) @ np.abs(q[j])).max() * abs(scale)
    assert heads * group == q.shape[0]
    return out, size, spread
