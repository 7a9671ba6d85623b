"""Launch configurations of the block-scaled e4m3 linear (``fp8_block_linear``).

A call's config follows from its M, N and K alone, by the rule of :func:`block_config`; there is no
table of tuned layers. ``BLOCK_TILES`` lists what the library compiles.
"""

from __future__ import annotations

from dataclasses import dataclass

BLOCK = 128
"""K and N of a weight's scale block, and K of an activation's."""


@dataclass(frozen=True)
class BlockConfig:
    """One launch: ``gemv_block`` (block_m rows x 16 columns per workgroup, ``num_warps`` waves share
    K), or ``gemm_block`` (block_m x block_n tiles, ``num_stages`` LDS stages, K in ``split_k`` slices that a
    second kernel adds)."""

    kernel: str
    block_m: int
    block_n: int
    split_k: int
    num_warps: int
    num_stages: int


BLOCK_TILES: tuple[tuple[str, int, int, int, int], ...] = (
    ("gemv_block", 16, 16, 8, 1), ("gemv_block", 64, 16, 4, 1),
    ("gemm_block", 256, 256, 8, 2), ("gemm_block", 256, 128, 8, 3), ("gemm_block", 128, 256, 8, 3),
    ("gemm_block", 128, 128, 4, 2), ("gemm_block", 128, 128, 8, 4), ("gemm_block", 64, 128, 8, 3),
    ("gemm_block", 64, 64, 4, 4),
)
"""(kernel, block_m, block_n, num_warps, num_stages) of every compiled kernel."""


def block_config(m: int, n: int, k: int) -> BlockConfig:
    """The launch of an M x N x K call."""
    if m <= 16:
        return BlockConfig("gemv_block", 16, 16, 1, 8, 1)
    nkb = -(-k // BLOCK)
    bm, bn, warps, stages = (64, 128, 8, 3) if m <= 64 else (128, 128, 8, 4) if m <= 512 else (256, 256, 8, 2)
    tiles = -(-m // bm) * -(-n // bn)
    split = max(1, min(256 // tiles, nkb // 4, 8))
    return BlockConfig("gemm_block", bm, bn, split, warps, stages)
