"""Launch configurations of the block-scaled e4m3 linear (``fp8_block_linear``).

A call's config follows from its M, N and K alone: of the compiled kernels and K splits, the one whose
modelled time is least. The models' constants were fitted to the measured times of every config on
about 4000 layers and row counts on MI355X (M 1 to 4096, weights of 16 KB to 136 MB, read from HBM): the
choice is 2.0% slower than the best compiled config on average, 5% at the 90th percentile. There is no
table of tuned layers.
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
class _Gemv:
    """Time in us: a start, the wave's share of blocks at ``block`` each, more where many waves share a CU,
    and the weight bytes at ``rate`` (bytes/us), ``again`` of them for every further row tile."""

    block_m: int
    num_warps: int
    start: float
    block: float
    crowd: float
    rate: float
    again: float

    def us(self, m: int, n: int, k: int) -> float:
        tiles_m = -(-m // self.block_m)
        groups = -(-n // 16) * tiles_m
        wave = -(-_blocks(k) // self.num_warps) * self.block
        compute = wave * (1 + groups * self.num_warps / (NUM_CUS * self.crowd))
        memory = n * k * (1 + self.again * (tiles_m - 1)) / self.rate
        return self.start + (compute**4 + memory**4) ** 0.25


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


_GEMV = (
    _Gemv(4, 8, 3.19, 0.610, 9.1, 4.41e6, 0.3),
    _Gemv(4, 4, 3.26, 0.363, 6.6, 4.28e6, 0.3),
    _Gemv(8, 4, 3.37, 0.377, 12.7, 3.50e6, 0.3),
    _Gemv(16, 4, 3.36, 0.505, 36.0, 2.79e6, 1.0),
)
_GEMM = (
    _Gemm(256, 256, 8, 2, 1, 6.00, 3.19, 1.296, 1.824, 3.92e6, 2.19, 6.95e6),
    _Gemm(128, 256, 8, 3, 1, 4.43, 2.86, 0.795, 1.060, 5.37e6, 2.42, 6.14e6),
    _Gemm(128, 128, 8, 4, 1, 3.11, 2.62, 0.567, 0.674, 5.35e6, 2.72, 5.31e6),
    _Gemm(64, 256, 8, 3, 1, 3.36, 2.34, 0.597, 0.720, 5.23e6, 2.59, 4.90e6),
    _Gemm(64, 64, 4, 4, 2, 2.44, 2.16, 0.384, 0.561, 5.73e6, 2.13, 3.24e6),
    _Gemm(32, 256, 4, 4, 1, 2.19, 2.97, 0.597, 0.666, 5.08e6, 2.68, 4.85e6),
    _Gemm(32, 128, 4, 4, 1, 1.79, 2.45, 0.417, 0.444, 6.03e6, 2.76, 4.44e6),
)
_GEMV_STAGES = 4
GEMV_MAX_M = 128
"""Row count up to which the gemv form is weighed (it reads the weight once per 16 rows)."""
_SPLITS = (1, 2, 3, 4, 6, 8, 12, 16)
_MAX_SPLIT_GROUPS = 700
"""Workgroups up to which K is split: past that the chip is full."""

BLOCK_TILES: tuple[tuple[str, int, int, int, int], ...] = tuple(
    [("gemv_block", g.block_m, 16, g.num_warps, _GEMV_STAGES) for g in _GEMV]
    + [("gemm_block", t.block_m, t.block_n, t.num_warps, t.num_stages) for t in _GEMM]
)
"""(kernel, block_m, block_n, num_warps, num_stages) of every compiled kernel."""


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


@functools.lru_cache(maxsize=4096)
def block_config(m: int, n: int, k: int) -> BlockConfig:
    """The launch of an M x N x K call: the least modelled time."""
    nkb = _blocks(k)
    rows = 4 if m <= 4 else 8 if m <= 8 else 16
    best: tuple[float, BlockConfig] | None = None
    if m <= GEMV_MAX_M:
        for g in _GEMV:
            if g.block_m == rows:
                us = g.us(m, n, k)
                if best is None or us < best[0]:
                    best = us, BlockConfig("gemv_block", rows, 16, 1, g.num_warps, _GEMV_STAGES)
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
