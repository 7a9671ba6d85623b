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


# ----------------------------------------------------------------------------- what the matrix instruction cuts

GROUP = 8
"""Consecutive k whose products the matrix instruction adds in one window."""


def cut_bound(x8: torch.Tensor, xs: torch.Tensor, w8: torch.Tensor, ws: torch.Tensor) -> np.ndarray:
    """How much the cuts of products can take from each output, whatever their signs: a product loses less than
    2^-13 of the power of two below the largest of its group of eight consecutive k, and the largest nothing."""
    n, k = w8.shape
    x, w = np.abs(e4m3_decode(bc.codes(x8)).astype(np.float64)), np.abs(e4m3_decode(bc.codes(w8)).astype(np.float64))
    scales = np.repeat(ws.double().numpy(), oblk.BLOCK, axis=0)[:n]
    total = np.zeros((x.shape[0], n))
    for k0 in range(0, k, GROUP):
        peak = (x[:, None, k0:k0 + GROUP] * w[None, :, k0:k0 + GROUP]).max(axis=2)
        unit = np.where(peak > 0, np.exp2(np.floor(np.log2(np.where(peak > 0, peak, 1.0))) - 13), 0.0)
        total += (GROUP - 1) * unit * xs.double().numpy()[:, k0 // 128, None] * scales[None, :, k0 // 128]
    return total


def hard_inputs(kind: str, m: int, n: int, k: int) -> tuple[torch.Tensor, ...]:
    """Operands of a linear whose products differ much in size inside a group of eight.

    ``outliers``: one channel of x in eight is 20 times the others, as hidden states have them. ``one sign``:
    the same without signs, so that every cut has one sign too. ``cancelling``: in each group two products of
    up to 2^17 that cancel, and six of one sign and about 2^3, which are all that is left of the sum."""
    g = bc.gen(kind, m, n, k)
    x, w = torch.randn((m, k), generator=g) * 7, torch.randn((n, k), generator=g) * 100
    x[:, ::GROUP] *= 20
    if kind == "one sign":
        x, w = x.abs(), w.abs()
    if kind == "cancelling":
        x, w = 2 + torch.rand((m, k), generator=g), 2 + 2 * torch.rand((n, k), generator=g)
        x[:, 0::GROUP] = x[:, 1::GROUP] = 448
        w[:, 0::GROUP] = 100 + 300 * torch.rand(w[:, 0::GROUP].shape, generator=g)
        w[:, 1::GROUP] = -w[:, 0::GROUP]
    nkb, nnb = -(-k // 128), -(-n // 128)
    xs = torch.exp2(torch.rand((m, nkb), generator=g) - 10)
    ws = torch.exp2(torch.rand((nnb, nkb), generator=g) - 12)
    f8 = torch.float8_e4m3fn
    return x.clamp(-448, 448).to(f8), xs, w.clamp(-448, 448).to(f8), ws


def remainder_residual(inputs: tuple[torch.Tensor, ...]) -> torch.Tensor:
    """The fp16 residual that leaves of a linear's outputs what their own rounding would hide."""
    x8, xs, w8, ws = inputs
    y = oblk.linear(bc.codes(x8), xs.numpy(), bc.codes(w8), ws.numpy())[0]
    assert np.abs(y).max() < 60000
    return torch.from_numpy(-y).to(torch.float16)


def check_remainder(out: torch.Tensor, inputs: tuple[torch.Tensor, ...], residual: torch.Tensor, what: str) -> None:
    """``out`` = the linear plus :func:`remainder_residual`: off by the cuts, the fp32 additions (a relative
    2^-23 of the sum of magnitudes each: sixteen groups, the blocks, two of scales, the residual's) and half
    an fp16 step of what is left."""
    x8, xs, w8, ws = inputs
    y, size, _ = oblk.linear(bc.codes(x8), xs.numpy(), bc.codes(w8), ws.numpy())
    r = residual.double().numpy()
    additions = 16 + -(-x8.shape[1] // 128) + 3
    carried = cut_bound(*inputs) + additions * 2 * bc.U32 * (size + np.abs(r))
    bound = carried + bc.HALF_STEP[torch.float16] * (np.abs(y + r) + carried) + 2.0**-25
    off = np.abs(out.detach().cpu().double().numpy() - (y + r))
    assert (off <= bound).all(), f"{what}: {int((~(off <= bound)).sum())} off, by up to {(off - bound).max():.3e} too much"
