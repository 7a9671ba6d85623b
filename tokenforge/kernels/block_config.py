"""Launch configurations of the block-scaled e4m3 linear (``fp8_block_linear``).

A call's config follows from its M, N and K alone. Few rows take the gemv form up to a weight size
(:func:`_gemv_tile`); else, of the compiled tiles and K splits, the one whose modelled time is least. The
limits and the model's constants come from the measured times of every config on about 6000 layers and
row counts on MI355X (M 1 to 4096, weights of 16 KB to 136 MB, read from HBM): the choice is 2 to 3% slower
than the best compiled config on average (M <= 4 1.5%, 9 to 16 rows 2.8%, 33 to 128 rows on small weights
4%). There is no table of tuned layers.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

BLOCK = 128
"""K and N of a weight's scale block, and K of an activation's."""
NUM_CUS = 256


@dataclass(frozen=True)
class BlockConfig:
    """One launch of ``tf_fp8_block_linear``.

    ========== ============================== ==============================================
    kernel     block_m / block_n              split_k / num_warps / num_stages
    ========== ============================== ==============================================
    gemv_block rows per workgroup (4 to 32)   1 / waves that share K / K blocks in flight
               / 16 columns                   per wave
    gemm_block tile rows / tile columns       K slices, added by a second kernel / waves /
                                              LDS stages
    ========== ============================== ==============================================
    """

    kernel: str
    block_m: int
    block_n: int
    split_k: int
    num_warps: int
    num_stages: int


@dataclass(frozen=True)
class _Gemm:
    """Time in us: a start; rounds of resident workgroups (``per_cu`` of them a CU), each ``fixed`` and a
    step per K block, ``alone`` to ``busy`` long as the CUs fill; the bytes at ``rate`` (bytes/us); for a
    K split the second kernel's ``reduce`` and the partial sums at ``reduce_rate``."""

    block_m: int
    block_n: int
    num_warps: int
    num_stages: int
    per_cu: int
    start: float
    fixed: float
    alone: float
    busy: float
    rate: float
    reduce: float
    reduce_rate: float

    def us(self, m: int, n: int, k: int, split: int) -> float:
        steps = -(-_blocks(k) // split)
        groups = -(-m // self.block_m) * -(-n // self.block_n) * split
        resident = NUM_CUS * self.per_cu

        def one_round(count: int) -> float:
            return self.fixed + steps * (self.alone + (self.busy - self.alone) * count / resident)

        rest = groups % resident
        compute = groups // resident * one_round(resident) + (one_round(rest) if rest else 0.0)
        memory = (n * k + m * k + 2 * m * n) / self.rate
        us = self.start + (compute**4 + memory**4) ** 0.25
        return us + self.reduce + 8 * m * n * split / self.reduce_rate if split > 1 else us


_GEMM = (
    _Gemm(256, 256, 8, 2, 1, 6.00, 3.19, 1.296, 1.824, 3.92e6, 2.19, 6.95e6),
    _Gemm(128, 256, 8, 3, 1, 4.43, 2.86, 0.795, 1.060, 5.37e6, 2.42, 6.14e6),
    _Gemm(128, 128, 8, 4, 1, 3.11, 2.62, 0.567, 0.674, 5.35e6, 2.72, 5.31e6),
    _Gemm(64, 256, 8, 3, 1, 3.36, 2.34, 0.597, 0.720, 5.23e6, 2.59, 4.90e6),
    _Gemm(64, 64, 4, 4, 2, 2.44, 2.16, 0.384, 0.561, 5.73e6, 2.13, 3.24e6),
    _Gemm(32, 256, 4, 4, 1, 2.19, 2.97, 0.597, 0.666, 5.08e6, 2.68, 4.85e6),
    _Gemm(32, 128, 4, 4, 1, 1.79, 2.45, 0.417, 0.444, 6.03e6, 2.76, 4.44e6),
)
_GEMV_TILES = ((4, 8, 4), (4, 4, 4), (8, 4, 4), (16, 4, 4), (32, 4, 2))
"""(block_m, num_warps, num_stages) of the gemv form."""
_SPLITS = (1, 2, 3, 4, 6, 8, 12, 16)
_MAX_SPLIT_GROUPS = 700
"""Workgroups up to which K is split: past that the chip is full."""

BLOCK_TILES: tuple[tuple[str, int, int, int, int], ...] = tuple(
    [("gemv_block", rows, 16, waves, stages) for rows, waves, stages in _GEMV_TILES]
    + [("gemm_block", t.block_m, t.block_n, t.num_warps, t.num_stages) for t in _GEMM]
)
"""(kernel, block_m, block_n, num_warps, num_stages) of every compiled kernel."""


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _gemv_tile(m: int, n: int, k: int) -> tuple[int, int, int] | None:
    """The gemv form's tile for a call, None where the gemm form is faster.

    The gemv form stages nothing: it wins while the weight is small and the rows are few, and loses where
    its reads of x (once per 16 columns) or of the weight (once per row tile) weigh more. MI355X, the two
    forms' best: 3584 x 3584 M = 7 6.2 us against 10.6, M = 20 8.4 against 11.0, M = 48 13.6 against 11.7;
    896 x 4864 M = 48 8.4 against 10.2, M = 128 10.6 against 11.6; 37888 x 3584 M = 12 43 against 29.6;
    3584 x 18944 M = 7 18.8 either way. Eight waves along K against four at M <= 4: 3584 x 18944 15.8 us
    against 17.9, 1152 x 896 3.9 against 3.7."""
    weight = n * k
    if m <= 4:
        return _GEMV_TILES[0] if k >= 2048 else _GEMV_TILES[1]
    if m <= 8:
        return _GEMV_TILES[2] if weight < 70e6 else None
    if m <= 16:
        return _GEMV_TILES[3] if weight < 24e6 else None
    if m <= 64 and weight < 5e6:
        return _GEMV_TILES[3]
    if (m <= 32 and weight < 16e6) or (m <= 128 and weight < 5e6) or (m <= 256 and weight < 1.5e6):
        return _GEMV_TILES[4]
    return None


@functools.lru_cache(maxsize=4096)
def block_config(m: int, n: int, k: int) -> BlockConfig:
    """The launch of an M x N x K call."""
    gemv = _gemv_tile(m, n, k)
    if gemv is not None:
        return BlockConfig("gemv_block", gemv[0], 16, 1, gemv[1], gemv[2])
    nkb = _blocks(k)
    best: tuple[float, BlockConfig] | None = None
    for t in _GEMM:
        tiles = -(-m // t.block_m) * -(-n // t.block_n)
        for split in _SPLITS:
            if split > 1 and (split > nkb // 2 or tiles > NUM_CUS or tiles * split > _MAX_SPLIT_GROUPS):
                break
            us = t.us(m, n, k, split)
            if best is None or us < best[0]:
                best = us, BlockConfig("gemm_block", t.block_m, t.block_n, split, t.num_warps, t.num_stages)
    assert best is not None
    return best[1]
