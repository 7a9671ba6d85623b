"""Launch configurations of the block-scaled e4m3 linear (``fp8_block_linear``).

A call's config follows from its M, N and K alone. Few rows take the gemv form up to a weight size
(:func:`_gemv_waves`); else, of the compiled tiles and K splits, the one whose modelled time is least. The
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
    gemv_block rows per workgroup (4, 8, 16)  1 / waves that share K / K blocks in flight
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
_GEMV_TILES = ((4, 8), (4, 4), (8, 4), (16, 4))  # rows, waves
_GEMV_STAGES = 4
_SPLITS = (1, 2, 3, 4, 6, 8, 12, 16)
_MAX_SPLIT_GROUPS = 700
"""Workgroups up to which K is split: past that the chip is full."""

BLOCK_TILES: tuple[tuple[str, int, int, int, int], ...] = tuple(
    [("gemv_block", rows, 16, waves, _GEMV_STAGES) for rows, waves in _GEMV_TILES]
    + [("gemm_block", t.block_m, t.block_n, t.num_warps, t.num_stages) for t in _GEMM]
)
"""(kernel, block_m, block_n, num_warps, num_stages) of every compiled kernel."""


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _gemv_waves(m: int, n: int, k: int) -> int:
    """Waves per workgroup of the gemv form, 0 where a tile is faster. The form reads the weight once per 16
    rows without staging x: on MI355X it wins while the weight is small (3584 x 3584 M = 7: 6.2 us against
    10.6 for the best tile; 896 x 4864 M = 12: 7.7 against 9.8) and loses on wide layers with more rows
    (37888 x 3584 M = 7: 29.6 against 25.1 to 31 over boxes, M = 12: 43 against 29.6). From K = 2048 on eight
    waves along K are faster than four at M <= 4 (3584 x 18944: 15.8 us against 17.9; 1152 x 896 the other
    way, 3.9 against 3.7)."""
    weight = n * k
    if m <= 4:
        return 8 if k >= 2048 else 4
    if m <= 8:
        return 4 if weight < 48e6 else 0
    if m <= 16:
        return 4 if weight < 24e6 else 0
    if m <= 32:
        return 4 if weight < 8e6 else 0
    return 4 if m <= 128 and weight * -(-m // 16) < 12e6 else 0


@functools.lru_cache(maxsize=4096)
def block_config(m: int, n: int, k: int) -> BlockConfig:
    """The launch of an M x N x K call."""
    waves = _gemv_waves(m, n, k)
    if waves:
        return BlockConfig("gemv_block", 4 if m <= 4 else 8 if m <= 8 else 16, 16, 1, waves, _GEMV_STAGES)
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
