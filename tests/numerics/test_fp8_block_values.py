"""FP8 with a scale per 128 on the GPU, further values and sizes: gates whose sigmoid leaves fp32's normal range;
codes that have to be numbers at every size; linears too long or wide for their usual launch; linears whose
products differ so much in size that the matrix instruction cuts some.

The norm's error: hidden squared, a tree of three and one of six levels, up to 64 sums of those in order, 1 / k,
its product and eps are 1 + 3 + 6 + 64 + 3 roundings of the mean, half as many of its root; root, quotient and
two products are four more: 43 roundings of 2^-24."""

from __future__ import annotations

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from oracle import fp8_block as oblk
from tests.numerics import block_cases as bc
from tests.numerics import block_codes
from tokenforge.kernels.block_config import BLOCK_TILES, BlockConfig
from tokenforge.kernels.hip.fp8_block import fp8_block_gemm

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
EPS = 1e-6
NORM_ERR = 43 * bc.U32


@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("k", [128, 130, 1000, 4864])
def test_silu_mul_of_gates_far_below_zero(k: int, group: int, device: torch.device) -> None:
    x = block_codes.far_gates(k)
    block_codes.check_far_gates(*ops.silu_mul_fp8_quant(x.to(device), group), x, group)


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize(("t", "k"), [(1, 1), (4, 7), (3, 130), (2, 1000), (17, 1296), (129, 264), (1030, 896), (1, 8200),
                                      (2, 18944), (1, 32767), (1, 32768)])
def test_codes_are_numbers(t: int, k: int, group: int, dtype: torch.dtype, device: torch.device) -> None:
    """Every code of every producer, the last ones of a ragged row and of each lane among them."""
    x, r, gu = (bc.rows(t, n, dtype, seed) for n, seed in ((k, 30), (k, 31), (2 * k, 32)))
    w = (torch.rand((k,), generator=bc.gen("w", k)) + 0.5).to(dtype)
    q, s = ops.fp8_quant(x.to(device), group)
    block_codes.check_codes(q, s, x.double().numpy(), 0.0, group, "fp8_quant")
    q, s = ops.silu_mul_fp8_quant(gu.to(device), group)
    block_codes.check_codes(q, s, oblk.silu_mul(gu.double().numpy()), block_codes.silu_err(gu), group, "silu")
    for res in (None, r):
        q, s, _ = ops.add_rmsnorm_fp8_quant(x.to(device), None if res is None else res.to(device), w.to(device), EPS,
                                            group)
        y = oblk.rmsnorm((x if res is None else x + res).double().numpy(), w.double().numpy(), EPS)
        block_codes.check_codes(q, s, y, NORM_ERR, group, "norm")


@pytest.mark.parametrize(("m", "n"), [(3, 300_000_000), ((1 << 30) + 5, 1)])
def test_linear_too_large_for_its_usual_launch(m: int, n: int, device: torch.device) -> None:
    """Where the gemv form, or the tile the time model prefers, would take 2^32 threads: outputs of the first,
    middle and last rows or columns. (The codes have one sign. With two groups of eight the cuts of either, 7 of
    2^-13 of its largest product, are within ``linear_bound``'s 7 sqrt(7) 2^-13 of the length all the same.)"""
    g = torch.Generator(device=device).manual_seed(m)
    x8, w8 = (torch.randint(0, 0x7F, (r, 16), generator=g, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
              for r in (m, n))
    xs = torch.rand((m, 1), generator=g, device=device) * 1e-2
    ws = torch.rand((-(-n // 128), 1), generator=g, device=device) * 1e-3
    y = ops.fp8_block_linear(x8, xs, w8, ws, None, torch.bfloat16, "hip")
    assert y.shape == (m, n)
    for r0 in sorted({0, m // 2, max(0, m - 40)}):
        for c0 in sorted({0, n // 256 * 128, (n - 1) // 128 * 128}):
            r, c = slice(r0, min(m, r0 + 40)), slice(c0, min(n, c0 + 128))
            inputs = (x8[r].cpu(), xs[r].cpu(), w8[c].cpu(), ws[c0 // 128:c0 // 128 + 1].cpu())
            bc.check_linear(y[r, c], inputs, f"{m}x{n} at {r0}, {c0}")


def _config(tile: tuple[str, int, int, int, int]) -> BlockConfig:
    kernel, bm, bn, warps, stages = tile
    return BlockConfig(kernel, bm, bn, 1, warps, stages)


@pytest.mark.parametrize("tile", BLOCK_TILES, ids=str)
def test_small_products_beside_a_large_one(tile, device: torch.device) -> None:  # type: ignore[no-untyped-def]
    """A product of 2^16 at one k, its negative 16 k further on (another group of eight), a small one at each
    other k in turn, a row of x each: in the large ones' groups 2^3 is kept whole and less may be lost, in the
    other groups 2^-7 is kept whole. (fp32's 24 bits hold 2^16 + 2^-7, but for 2^16 + 2^-8 it takes 25.)"""
    k, at = 128, 37
    back = at + 16
    others = [j for j in range(k) if j not in (at, back)]
    for e in (6, 3, 2, 0, -7, -8):
        x = torch.zeros((len(others), k))
        w = torch.ones((3, k))
        x[:, at] = x[:, back] = 256.0
        w[:, at], w[:, back] = 256.0, -256.0
        small = 2.0 ** (e / 2 if e % 2 == 0 else (e - 1) / 2)
        for r, j in enumerate(others):
            x[r, j] = small
        w[:, others] = 2.0**e / small
        f8 = torch.float8_e4m3fn
        assert torch.equal(x.to(f8).float(), x) and torch.equal(w.to(f8).float(), w)
        y = fp8_block_gemm(x.to(f8).to(device), torch.ones((len(others), 1), device=device), w.to(f8).to(device),
                           torch.ones((1, 1), device=device), _config(tile)).cpu()
        for r, j in enumerate(others):
            near = j // 8 in (at // 8, back // 8)
            ok = (y[r] == 2.0**e) | ((y[r] >= 0) & (y[r] <= 2.0**e) if (near and e < 3) or e < -7 else False)
            assert bool(ok.all()), (e, j, y[r])


@pytest.mark.parametrize("kind", ["outliers", "one sign", "cancelling"])
@pytest.mark.parametrize("tile", BLOCK_TILES, ids=str)
def test_linear_of_products_far_apart(tile, kind: str, device: torch.device) -> None:  # type: ignore[no-untyped-def]
    inputs = block_codes.hard_inputs(kind, 21, 150, 1040)
    residual = block_codes.remainder_residual(inputs)
    y = fp8_block_gemm(*(t.to(device) for t in inputs), _config(tile), None, torch.float16, residual.to(device))
    block_codes.check_remainder(y, inputs, residual, f"{kind} {tile}")


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize(("n", "with_bias", "with_residual"), [(8000, True, True), (8000, False, True), (8000, True, False),
                                                               (8001, True, True)])
def test_outputs_past_the_caches(n: int, with_bias: bool, with_residual: bool, dtype: torch.dtype,
                                 device: torch.device) -> None:
    """Outputs above 32 MB of the largest tile, which are stored past the L2s: bias, residual and rows whose
    length takes no 16-byte store."""
    m, k = 2201, 256
    inputs = bc.linear_inputs(m, n, k, seed=50)
    g = bc.gen("past", n)
    bias = (torch.randn((n,), generator=g) * 4).to(dtype) if with_bias else None
    residual = (torch.randn((m, n), generator=g) * 4).to(dtype) if with_residual else None
    y = fp8_block_gemm(*(t.to(device) for t in inputs), BlockConfig("gemm_block", 256, 256, 1, 8, 2),
                       None if bias is None else bias.to(device), dtype,
                       None if residual is None else residual.to(device))
    bc.check_linear(y, inputs, f"{n} {dtype}", bias, residual)
