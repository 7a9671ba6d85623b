"""Launch configurations of the block-scaled e4m3 linear (``fp8_block_linear``).

A call's config follows from its M, N and K alone: of the compiled tiles and K splits, the one whose
modelled time is least (up to four rows always the gemv form, by :func:`_one_tile`). The models'
constants are fitted to measured times of every config on MI355X, weights read from HBM: 4560 layers and row
counts (M 5 to 2500, weights of 16 KB to 136 MB). There the choice is 0.6% slower on average than the
best compiled config (99 of 100 within 9%); on others, 0.3% at M 2000 to 9000 and 0.8% at M 1 to 2500, of
which 2.3% up to four rows. There is no table of tuned layers. ``bench_probes/block_choice.py`` times every
config of a call, the data of such a fit (the small decoder's down projection at M = 16 loses most: 7.9 us
against 6.4 of the four-row gemv form, which the rule keeps to four rows).
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
    """Time in us: a start; rounds of one workgroup a CU, each ``fixed`` and a step per K block, ``alone`` to
    ``busy`` long as the CUs fill; the bytes at ``rate`` (bytes/us); for a
    K split the second kernel's ``reduce`` and the partial sums at ``reduce_rate``."""

    block_m: int
    block_n: int
    num_warps: int
    num_stages: int
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

        def one_round(count: int) -> float:
            return self.fixed + steps * (self.alone + (self.busy - self.alone) * count / NUM_CUS)

        rest = groups % NUM_CUS
        compute = groups // NUM_CUS * one_round(NUM_CUS) + (one_round(rest) if rest else 0.0)
        memory = (n * k + m * k + 2 * m * n) / self.rate
        us = self.start + (compute**4 + memory**4) ** 0.25
        return us + self.reduce + 8 * m * n * split / self.reduce_rate if split > 1 else us


@dataclass(frozen=True)
class _Gemv:
    """Time in us: a start; rounds of one workgroup a CU, each ``fixed`` and a ``step`` per K block of a
    wave; the bytes at ``rate`` (bytes/us). Considered from ``fewest`` to ``most`` rows."""

    fewest: int
    most: int
    block_m: int
    num_warps: int
    num_stages: int
    start: float
    fixed: float
    step: float
    rate: float

    def us(self, m: int, n: int, k: int) -> float:
        rounds = -(-(-(-m // self.block_m) * -(-n // 16)) // NUM_CUS)
        compute = rounds * (self.fixed + -(-_blocks(k) // self.num_warps) * self.step)
        memory = (n * k + m * k + 2 * m * n) / self.rate
        return self.start + (compute**4 + memory**4) ** 0.25


_GEMM = (
    _Gemm(256, 256, 8, 2, 4.92, 6.00, 1.214, 1.791, 4.82e6, 1.35, 8.16e6),
    _Gemm(128, 256, 8, 3, 3.22, 4.91, 0.747, 1.022, 6.72e6, 1.78, 6.46e6),
    _Gemm(128, 128, 8, 4, 2.93, 3.13, 0.522, 0.664, 7.32e6, 2.08, 4.87e6),
    _Gemm(64, 256, 8, 3, 2.76, 3.08, 0.554, 0.733, 6.31e6, 1.98, 4.48e6),
    _Gemm(64, 128, 8, 3, 2.47, 3.59, 0.286, 0.386, 5.77e6, 1.97, 4.04e6),
    _Gemm(64, 64, 8, 4, 2.40, 2.85, 0.242, 0.310, 7.68e6, 2.06, 3.71e6),
    _Gemm(32, 128, 4, 4, 2.12, 2.31, 0.385, 0.487, 7.22e6, 2.28, 4.59e6),
    _Gemm(32, 64, 8, 3, 2.10, 3.07, 0.126, 0.175, 5.47e6, 2.12, 3.27e6),
)
_GEMV = (
    _Gemv(5, 8, 8, 4, 4, 3.16, 0.116, 0.339, 5.63e6),
    _Gemv(9, 300, 16, 4, 4, 3.09, 0.065, 0.489, 4.94e6),
    _Gemv(17, 300, 32, 4, 2, 3.05, 0.000, 0.684, 2.90e6),
)
_ONE_TILES = ((4, 8, 4), (4, 4, 4))
"""(block_m, num_warps, num_stages) of the gemv form up to four rows."""
_SPLITS = (1, 2, 3, 4, 6, 8, 12, 16)
_MAX_SPLIT_GROUPS = 700
"""Workgroups up to which K is split: past that the chip is full."""
_MAX_THREADS = 0xFFFFFFFF
"""Of one launch."""

BLOCK_TILES: tuple[tuple[str, int, int, int, int], ...] = tuple(
    [("gemv_block", rows, 16, waves, stages) for rows, waves, stages in _ONE_TILES]
    + [("gemv_block", t.block_m, 16, t.num_warps, t.num_stages) for t in _GEMV]
    + [("gemm_block", t.block_m, t.block_n, t.num_warps, t.num_stages) for t in _GEMM]
)
"""(kernel, block_m, block_n, num_warps, num_stages) of every compiled kernel."""


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _one_tile(k: int) -> tuple[int, int, int]:
    """The gemv form's tile up to four rows. Eight waves along K against four, us on MI355X: 3584 x 18944
    15.8 against 17.9, 1152 x 896 3.9 against 3.7."""
    return _ONE_TILES[0] if k >= 2048 else _ONE_TILES[1]


@functools.lru_cache(maxsize=4096)
def block_config(m: int, n: int, k: int) -> BlockConfig:
    """The launch of an M x N x K call."""
    rows, waves, stages = _one_tile(k)
    if m <= 4 and -(-n // 16) * 64 * waves <= _MAX_THREADS:
        return BlockConfig("gemv_block", rows, 16, 1, waves, stages)
    nkb = _blocks(k)
    best: tuple[float, BlockConfig] | None = None
    for v in _GEMV:
        if v.fewest <= m <= v.most and -(-n // 16) * 64 * v.num_warps <= _MAX_THREADS:
            us = v.us(m, n, k)
            if best is None or us < best[0]:
                best = us, BlockConfig("gemv_block", v.block_m, 16, 1, v.num_warps, v.num_stages)
    for t in _GEMM:
        tiles = -(-m // t.block_m) * -(-n // t.block_n)
        for split in _SPLITS:
            if split > 1 and (split > nkb // 2 or tiles > NUM_CUS or tiles * split > _MAX_SPLIT_GROUPS):
                break
            # The first tile, the largest, takes the fewest threads: where it takes too many, all do.
            if best is not None and tiles * split * 64 * t.num_warps > _MAX_THREADS:
                break
            us = t.us(m, n, k, split)
            if best is None or us < best[0]:
                best = us, BlockConfig("gemm_block", t.block_m, t.block_n, split, t.num_warps, t.num_stages)
    assert best is not None
    return best[1]
