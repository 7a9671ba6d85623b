"""More of the inputs and checks of FP8 with a scale per 128: codes that have to be numbers, and gates far
below zero."""

from __future__ import annotations

import numpy as np
import torch

from oracle import fp8_block as oblk
from oracle.reference import e4m3_decode
from tests.numerics import block_cases as bc


def check_codes(q: torch.Tensor, s: torch.Tensor, y: np.ndarray, err: np.ndarray | float, group_size: int,
                what: str) -> None:
    """:func:`block_cases.check_codes` of finite ``y``, where no code and no scale may be a NaN (a comparison
    that asks for an excess over the bound lets a NaN through)."""
    assert np.isfinite(y).all(), what
    bad = ~np.isfinite(e4m3_decode(bc.codes(q)).astype(np.float64))
    assert not bad.any(), f"{what}: {int(bad.sum())} codes are NaN, first at {np.argwhere(bad)[0]}"
    assert bool(torch.isfinite(s).all()), f"{what}: a scale is not finite"
    bc.check_codes(q, s, y, err, group_size, what)


def silu_err(x: torch.Tensor) -> np.ndarray:
    """Relative error of ``silu(gate) * up`` in fp32: 8 roundings, and the exponential's argument, whose
    rounding (with that of its constant) grows with the gate."""
    gate = np.abs(x.double().numpy()[:, : x.shape[1] // 2])
    return (8 + 2 * gate) * bc.U32


def far_gates(k: int) -> torch.Tensor:
    """bf16 ``[gate | up]`` rows ``[20, 2 k]``: gates in windows of four from -72 down to -150 (row 19: down to
    -2000), ups of 1e38 to 3e38 and both signs, so the product is some 1e9 at -72, 1 at -92 and below
    the smallest scale's codes from -116 on."""
    g = bc.gen("far", k)
    top = -72.0 - 4.0 * torch.arange(20)[:, None]
    gate = top - 4.0 * torch.rand((20, k), generator=g)
    gate[19] = -150.0 - 1850.0 * torch.rand((k,), generator=g)
    up = (1.0 + 2.0 * torch.rand((20, k), generator=g)) * 1e38
    up[torch.rand((20, k), generator=g) < 0.5] *= -1.0
    return torch.cat([gate, up], 1).to(torch.bfloat16)


def check_far_gates(q: torch.Tensor, s: torch.Tensor, x: torch.Tensor, group: int) -> None:
    y = oblk.silu_mul(x.double().numpy())
    check_codes(q, s, y, silu_err(x), group, f"gates below -72, group {group}")
    largest = np.abs(e4m3_decode(bc.codes(q))).max(axis=1)
    # Rows 0 to 6 (gates down to -100) have scales above the smallest one, rows 7 to 9 codes at the smallest.
    assert (largest[:7] == 448).all() and (largest[7:10] > 0).all() and largest[19] == 0
