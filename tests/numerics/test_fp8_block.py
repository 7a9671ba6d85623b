"""FP8 with a scale per 128 on the GPU: the quantizers and the block-scaled linear against their
definitions in 64 bits (``oracle/fp8_block.py``), at the sizes, layouts and values where they can go wrong.

Bounds are derived beside ``block_cases.check_codes`` and ``linear_bound``. The errors handed to them:
``fp8_quant`` reads its values exactly; SiLU * up has an exponential, an addition, a division and a
product, 8 roundings, and the exponential's argument, whose rounding grows with the gate; the norm has a
sum of squares (every addition a rounding, at most 24 levels of a tree and runs of 64), its root and
three products.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.library import opcheck

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from oracle import fp8_block as oblk
from tests.numerics import block_cases as bc
from tokenforge.kernels import host
from tokenforge.kernels.block_config import BLOCK_TILES, BlockConfig, block_config
from tokenforge.kernels.hip.fp8_block import fp8_block_gemm
from tokenforge.kernels.metrics import KERNEL_CALLS

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
EPS = 1e-6
NORM_ERR = 32 * bc.U32
SIZES = [(1, 3584), (3, 896), (2, 128), (5, 1), (4, 7), (3, 130), (2, 1000), (17, 1296), (1, 18944), (129, 264)]


def _silu_err(x: torch.Tensor) -> np.ndarray:
    gate = np.abs(x.double().numpy()[:, : x.shape[1] // 2])
    return (8 + 2 * gate) * bc.U32


# ----------------------------------------------------------------------------- quantizers


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize(("t", "k"), SIZES)
def test_quant(t: int, k: int, group: int, dtype: torch.dtype, device: torch.device) -> None:
    x = bc.rows(t, k, dtype)
    q, s = ops.fp8_quant(x.to(device), group)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    bc.check_codes(q, s, x.double().numpy(), 0.0, group, "fp8_quant")
    # The same values as torch's expression, bit for bit, scales and codes.
    qh, sh = host.block_quant(x.float(), group)
    assert torch.equal(s.cpu(), sh)
    assert np.array_equal(bc.codes(q), bc.codes(qh))


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize(("t", "k"), SIZES)
def test_silu_mul_quant(t: int, k: int, group: int, dtype: torch.dtype, device: torch.device) -> None:
    x = bc.rows(t, 2 * k, dtype, seed=1)
    q, s = ops.silu_mul_fp8_quant(x.to(device), group)
    bc.check_codes(q, s, oblk.silu_mul(x.double().numpy()), _silu_err(x), group, "silu_mul_fp8_quant")


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("with_residual", [True, False])
@pytest.mark.parametrize(("t", "k"), [*SIZES, (1, 32768), (2, 8200), (3, 32767), (2100, 896)])
def test_add_rmsnorm_quant(t: int, k: int, with_residual: bool, group: int, dtype: torch.dtype,
                           device: torch.device) -> None:
    x, r = bc.rows(t, k, dtype, seed=2), bc.rows(t, k, dtype, seed=3)
    w = (torch.rand((k,), generator=bc.gen("w", k)) + 0.5).to(dtype)
    q, s, hidden = ops.add_rmsnorm_fp8_quant(x.to(device), r.to(device) if with_residual else None, w.to(device), EPS,
                                             group)
    h = x + r if with_residual else x
    if with_residual:
        assert torch.equal(hidden.cpu(), h)
    else:
        assert hidden.shape == (0,)
    bc.check_codes(q, s, oblk.rmsnorm(h.double().numpy(), w.double().numpy(), EPS), NORM_ERR, group, "norm")


def test_a_row_does_not_depend_on_its_batch(device: torch.device) -> None:
    for t, k in ((2500, 896), (2500, 3584), (300, 8192)):
        x, r = bc.rows(t, k, torch.float16, 4).to(device), bc.rows(t, k, torch.float16, 5).to(device)
        w = torch.ones(k, dtype=torch.float16, device=device)
        for group in (128, 0):
            whole = ops.add_rmsnorm_fp8_quant(x, r, w, EPS, group)
            for at in (0, 1, t - 1):
                one = ops.add_rmsnorm_fp8_quant(x[at:at + 1], r[at:at + 1], w, EPS, group)
                for a, b in zip(one, whole):
                    assert np.array_equal(bc.codes(a), bc.codes(b[at:at + 1]))


def test_quant_of_zeros_and_of_the_largest_values(device: torch.device) -> None:
    for dtype in bc.DTYPES:
        x = torch.zeros((3, 256), dtype=dtype)
        x[1, :128] = torch.finfo(dtype).max
        x[1, 128:] = torch.finfo(dtype).smallest_normal
        x[2] = -torch.finfo(dtype).max
        for group in (128, 0):
            q, s = ops.fp8_quant(x.to(device), group)
            qh, sh = host.block_quant(x.float(), group)
            assert torch.equal(s.cpu(), sh) and np.array_equal(bc.codes(q), bc.codes(qh))


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nan_and_infinity_stay_in_their_block_or_row(bad: float, dtype: torch.dtype, device: torch.device) -> None:
    x = bc.rows(3, 384, dtype, seed=6)
    x[1, 130] = bad
    x[1, 131] = 0.0
    w = torch.ones(384, dtype=dtype)
    for group in (128, 0):
        q, s = ops.fp8_quant(x.to(device), group)
        qh, sh = host.block_quant(x.float(), group)
        assert torch.equal(torch.nan_to_num(s.cpu(), 7.0, 9.0), torch.nan_to_num(sh, 7.0, 9.0))
        assert torch.equal(torch.nan_to_num(q.float().cpu(), 999.0), torch.nan_to_num(qh.float(), 999.0))
        both = torch.cat([x, x], 1).to(device)
        q, s = ops.silu_mul_fp8_quant(both, group)
        qh, sh = host.silu_mul_block_quant(both.cpu(), group)
        hit = torch.zeros(q.shape, dtype=torch.bool)
        hit[1, 128:256 if group else 384] = True
        hit[1, :128] |= group == 0
        assert torch.equal(torch.isfinite(q.float().cpu())[~hit], torch.ones_like(hit)[~hit])
        assert torch.equal(torch.isnan(q.float().cpu()), torch.isnan(qh.float()))
        q, s, _ = ops.add_rmsnorm_fp8_quant(x.to(device), None, w.to(device), EPS, group)
        qh, sh, _ = host.add_rmsnorm_block_quant(x, None, w, EPS, group)
        assert torch.equal(torch.isnan(q.float().cpu()), torch.isnan(qh.float()))
        assert torch.equal(torch.isnan(s.cpu()), torch.isnan(sh))
        assert not torch.isnan(q.float()[0]).any() and not torch.isnan(q.float()[2]).any()


def test_quantizers_take_any_layout(device: torch.device) -> None:
    """Leading dimensions, rows further apart than their length, unaligned and transposed views, rows read
    twice: the result of a contiguous copy."""
    base = bc.rows(40, 2000, torch.float16, seed=7).to(device)
    views = [base[:24].reshape(2, 3, 4, 2000)[..., :512], base[:, 8:264], base[:, 3:259], base[::2, :130],
             base[:, :300].t(), base[:1, :256].expand(5, 256), base[:9, 1:2]]
    for v in views:
        c = v.contiguous()
        w = torch.ones(v.shape[-1], dtype=v.dtype, device=device)
        pairs = [(ops.fp8_quant(v, 128), ops.fp8_quant(c, 128)),
                 (ops.add_rmsnorm_fp8_quant(v, v, w, EPS, 0), ops.add_rmsnorm_fp8_quant(c, c, w, EPS, 0))]
        if v.shape[-1] % 2 == 0:
            pairs.append((ops.silu_mul_fp8_quant(v, 128), ops.silu_mul_fp8_quant(c, 128)))
        for got, want in pairs:
            for a, b in zip(got, want):
                assert a.shape == b.shape and np.array_equal(bc.codes(a), bc.codes(b))
    assert ops.fp8_quant(views[0], 128)[1].shape == (2, 3, 4, 4)


def test_row_scales_feed_w4a8_linear(device: torch.device) -> None:
    """group_size 0 gives what ``w4a8_linear`` reads."""
    from tests.numerics import cases

    w = cases.on_device(cases.layer_weights(256, 512, 0), device)
    x = cases.activations(5, 512, 0).to(device)
    q, s = ops.fp8_quant(x, 0)
    y = ops.w4a8_linear(q, s, w.qweight_t, w.scales, w.qzeros, None, 128, "hip")
    a = (q.float() * s).to(torch.float16)
    want = ops.w4a16_linear(a, w.qweight_t, w.scales, w.qzeros, None, 128, "hip")
    assert float((y.float() - want.float()).abs().max() / want.float().abs().max()) <= 2e-3


# ----------------------------------------------------------------------------- linear


def _to(device: torch.device, tensors):  # type: ignore[no-untyped-def]
    return tuple(t.to(device) for t in tensors)


def _config(tile: tuple[str, int, int, int, int], split: int = 1) -> BlockConfig:
    kernel, bm, bn, warps, stages = tile
    return BlockConfig(kernel, bm, bn, split, warps, stages)


LINEAR_SIZES = [(1, 16, 128), (1, 1, 16), (2, 130, 144), (15, 257, 1296), (16, 512, 256), (17, 129, 640), (65, 96, 272),
                (130, 300, 1024), (257, 385, 400), (520, 515, 128)]


@pytest.mark.parametrize(("m", "n", "k"), LINEAR_SIZES)
@pytest.mark.parametrize("tile", BLOCK_TILES, ids=str)
def test_linear_of_every_compiled_config(tile, m: int, n: int, k: int, device: torch.device) -> None:  # type: ignore[no-untyped-def]
    inputs = bc.linear_inputs(m, n, k)
    d = _to(device, inputs)
    for split in ((1,) if tile[0] == "gemv_block" else (1, 2, 5)):
        cfg = _config(tile, split)
        y = fp8_block_gemm(*d, cfg)
        bc.check_linear(y, inputs, f"{cfg} {m}x{n}x{k}")
        assert torch.equal(y, fp8_block_gemm(*d, cfg)), "reruns differ"


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize(("m", "n", "k"), [(1, 4608, 896), (3, 1000, 1296), (7, 896, 4864), (33, 1160, 512),
                                           (48, 2304, 896), (200, 1000, 1296), (333, 896, 2048), (1000, 640, 896)])
def test_linear_with_bias_and_residual(m: int, n: int, k: int, dtype: torch.dtype, device: torch.device) -> None:
    inputs = bc.linear_inputs(m, n, k, seed=1)
    g = bc.gen("extras", m, n)
    bias, res = (torch.randn((n,), generator=g) * 4).to(dtype), (torch.randn((m, n), generator=g) * 4).to(dtype)
    d, b, r = _to(device, inputs), bias.to(device), res.to(device)
    KERNEL_CALLS.reset()
    bc.check_linear(ops.fp8_block_linear(*d, None, dtype, "hip"), inputs, "plain")
    bc.check_linear(ops.fp8_block_linear(*d, b, dtype, "hip"), inputs, "bias", bias)
    bc.check_linear(ops.fp8_block_linear(*d, None, dtype, "hip", "residual", r), inputs, "residual", None, res)
    y = ops.fp8_block_linear(*d, b, dtype, "hip", "residual", r)
    bc.check_linear(y, inputs, "both", bias, res)
    assert torch.equal(y, fp8_block_gemm(*d, block_config(m, n, k), b, dtype, r))
    assert sum(KERNEL_CALLS.value(kernel=f, bucket=bkt) for f in ("hip_gemv", "hip_gemm")
               for bkt in ("1", "4", "8", "64", "256", "512", "1024")) == 4


def test_linear_of_nan_codes(device: torch.device) -> None:
    """A NaN code of x makes its row NaN, one of the weight its column, and nothing else."""
    for m in (1, 5, 40, 300):
        x8, xs, w8, ws = _to(device, bc.linear_inputs(m, 300, 272, seed=2))
        y = ops.fp8_block_linear(x8, xs, w8, ws, None, torch.float16, "hip")
        xn, wn = x8.view(torch.uint8).clone(), w8.view(torch.uint8).clone()
        xn[m // 2, 271], wn[137, 5] = 0x7F, 0xFF
        z = ops.fp8_block_linear(xn.view(torch.float8_e4m3fn), xs, wn.view(torch.float8_e4m3fn), ws, None,
                                 torch.float16, "hip")
        hit = torch.zeros((m, 300), dtype=torch.bool, device=device)
        hit[m // 2], hit[:, 137] = True, True
        assert bool(torch.isnan(z[hit]).all()) and torch.equal(z[~hit], y[~hit])


def test_linear_does_not_read_past_its_rows(device: torch.device) -> None:
    """K that ends inside a block, N inside a tile, M inside a tile: NaN codes right behind the rows' ends
    and behind the last row take no part."""
    for m, n, k in ((1, 20, 144), (9, 100, 272), (40, 130, 400), (300, 270, 656)):
        inputs = _to(device, bc.linear_inputs(m, n, k, seed=3))
        want = ops.fp8_block_linear(*inputs, None, torch.float16, "hip")
        x8, xs, w8, ws = inputs
        xb = torch.full((m + 3, k + 64), 0x7F, dtype=torch.uint8, device=device)
        wb = torch.full((n + 3, k + 64), 0x7F, dtype=torch.uint8, device=device)
        xb[:m, :k], wb[:n, :k] = x8.view(torch.uint8), w8.view(torch.uint8)
        sb = torch.full((m + 3, xs.shape[1] + 2), float("nan"), device=device)
        sb[:m, : xs.shape[1]] = xs
        tb = torch.full((ws.shape[0] + 1, ws.shape[1] + 2), float("nan"), device=device)
        tb[: ws.shape[0], : ws.shape[1]] = ws
        f8 = torch.float8_e4m3fn
        got = ops.fp8_block_linear(xb.view(f8)[:m, :k], sb[:m, : xs.shape[1]], wb.view(f8)[:n, :k],
                                   tb[: ws.shape[0], : ws.shape[1]], None, torch.float16, "hip")
        assert torch.equal(got, want)


def test_linear_takes_any_layout(device: torch.device) -> None:
    """Leading dimensions, transposed, unaligned and repeated operands: the result of contiguous copies."""
    m, n, k = 12, 200, 272
    x8, xs, w8, ws = _to(device, bc.linear_inputs(m, n, k, seed=4))
    res = torch.randn((m, n), generator=bc.gen("res")).to(torch.float16).to(device)
    want = ops.fp8_block_linear(x8, xs, w8, ws, None, torch.float16, "hip", "residual", res)
    got = ops.fp8_block_linear(x8.view(2, 2, 3, k), xs.view(2, 2, 3, -1), w8, ws, None, torch.float16, "hip",
                               "residual", res.view(2, 2, 3, n))
    assert got.shape == (2, 2, 3, n) and torch.equal(got.view(m, n), want)
    f8, u8 = torch.float8_e4m3fn, torch.uint8
    xt = x8.view(u8).t().contiguous().t().view(f8)
    wu = torch.zeros((n, k + 5), dtype=u8, device=device)
    wu[:, 5:] = w8.view(u8)
    got = ops.fp8_block_linear(xt, xs.t().contiguous().t(), wu[:, 5:].view(f8), ws.t().contiguous().t(), None,
                               torch.float16, "hip", "residual", res.t().contiguous().t())
    assert torch.equal(got, want)
    one = ops.fp8_block_linear(x8[:1].view(u8).expand(m, k).view(f8), xs[:1].expand(m, -1), w8, ws, None,
                               torch.float16, "hip", "residual", res[:1].expand(m, n))
    first = ops.fp8_block_linear(x8[:1], xs[:1], w8, ws, None, torch.float16, "hip", "residual", res[:1])
    bc.check_linear(one, (x8[:1].cpu().view(u8).expand(m, k).contiguous().view(f8), xs[:1].cpu().expand(m, -1),
                          w8.cpu(), ws.cpu()), "repeated rows", None, res[:1].cpu().expand(m, n))
    bc.check_linear(first, (x8[:1].cpu(), xs[:1].cpu(), w8.cpu(), ws.cpu()), "first row", None, res[:1].cpu())


@pytest.mark.parametrize("m", [1, 3, 7, 12, 40])
def test_linear_of_more_than_64_blocks_a_wave(m: int, device: torch.device) -> None:
    """K so long that a wave runs out of its 64 weight scales and loads the next."""
    n, k = 40, 66064
    inputs = bc.linear_inputs(m, n, k, seed=7)
    d = _to(device, inputs)
    bc.check_linear(ops.fp8_block_linear(*d, None, torch.bfloat16, "hip"), inputs, "op")
    for tile in BLOCK_TILES:
        if tile[0] == "gemv_block" or tile[1] <= 64:
            bc.check_linear(fp8_block_gemm(*d, _config(tile)), inputs, str(tile))


def test_rows_far_apart(device: torch.device) -> None:
    """Rows of codes 5 MB apart and of scales 2^20 elements apart are copied; the result is that of near ones."""
    x8, xs, w8, ws = _to(device, bc.linear_inputs(3, 40, 256, seed=8))
    want = ops.fp8_block_linear(x8, xs, w8, ws, None, torch.float16, "hip")
    far = torch.full((3, 5 << 20), 0x7F, dtype=torch.uint8, device=device)
    far[:, :256] = x8.view(torch.uint8)
    sfar = torch.full((3, 1 << 20), float("nan"), device=device)
    sfar[:, :2] = xs
    got = ops.fp8_block_linear(far.view(torch.float8_e4m3fn)[:, :256], sfar[:, :2], w8, ws, None, torch.float16, "hip")
    assert torch.equal(got, want)


def test_calls_on_two_streams_at_once(device: torch.device) -> None:
    """K-split calls (each with a workspace of its own) that overlap on two streams."""
    sets = [_to(device, bc.linear_inputs(64, 512, 8192, seed=s)) for s in (9, 10)]
    cfg = BlockConfig("gemm_block", 64, 64, 8, 8, 4)
    want = [fp8_block_gemm(*d, cfg) for d in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got: list[list[torch.Tensor]] = [[], []]
    for _ in range(20):
        for i, (d, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(fp8_block_gemm(*d, cfg))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize(("m", "n", "k"), [(3, 135000, 16384), (140000, 48, 16384), (70000, 35000, 128)])
def test_linear_past_32_bit_offsets(m: int, n: int, k: int, device: torch.device) -> None:
    """x8, the weight and the output beyond 2 GiB: the first and last rows and columns are those of a small
    call on them."""
    g = torch.Generator(device=device).manual_seed(m)

    def codes8(r: int) -> torch.Tensor:
        out = torch.empty((r, k), dtype=torch.uint8, device=device)
        for at in range(0, r, 16384):
            part = out[at:at + 16384]
            part.copy_((torch.randn(part.shape, generator=g, device=device, dtype=torch.float16) * 100)
                       .clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        return out.view(torch.float8_e4m3fn)

    x8, w8 = codes8(m), codes8(n)
    xs = torch.rand((m, k // 128), generator=g, device=device) * 1e-2
    ws = torch.rand((-(-n // 128), k // 128), generator=g, device=device) * 1e-3
    y = ops.fp8_block_linear(x8, xs, w8, ws, None, torch.bfloat16, "hip")
    rows = sorted({0, 1, m // 2, m - 1})
    n0 = n // 128 * 128 - 128 if n > 256 else 0
    for cols in (slice(0, min(n, 256)), slice(n0, n)):
        inputs = (x8.view(torch.uint8)[rows].view(torch.float8_e4m3fn).cpu(),
                  xs[rows].cpu(), w8[cols].cpu(), ws[cols.start // 128:-(-cols.stop // 128)].cpu())
        bc.check_linear(y[rows][:, cols], inputs, f"{m}x{n}x{k} {cols}")


@pytest.mark.parametrize("t", [(1 << 21) + 70, (1 << 26) + 5])
def test_quantizers_of_more_rows_than_one_launch_takes(t: int, device: torch.device) -> None:
    """A row's result is that of a call on few rows around it."""
    g = torch.Generator(device=device).manual_seed(t)
    x = torch.randn((t, 8), generator=g, device=device, dtype=torch.float16)
    w = torch.rand(8, generator=g, device=device, dtype=torch.float16)
    at = [slice(0, 40), slice((1 << 21) - 20, (1 << 21) + 20), slice(t - 40, t)]
    for group in (128, 0):
        calls = [lambda v: ops.fp8_quant(v, group), lambda v: ops.silu_mul_fp8_quant(v, group),
                 lambda v: ops.add_rmsnorm_fp8_quant(v, v, w, 1e-6, group)]
        for i, call in enumerate(calls):
            got = call(x)
            for s in at:
                for a, b in zip(got, call(x[s])):
                    assert torch.equal(a[s].view(torch.uint8), b.view(torch.uint8)), (i, group, s)
            del got


def test_empty_calls(device: torch.device) -> None:
    e8 = torch.empty((0, 256), dtype=torch.float8_e4m3fn, device=device)
    _, _, w8, ws = _to(device, bc.linear_inputs(1, 130, 256))
    y = ops.fp8_block_linear(e8, torch.empty((0, 2), device=device), w8, ws, None, torch.bfloat16, "hip")
    assert y.shape == (0, 130) and y.dtype == torch.bfloat16
    x = torch.empty((2, 0, 256), dtype=torch.float16, device=device)
    q, s = ops.fp8_quant(x, 128)
    assert q.shape == (2, 0, 256) and s.shape == (2, 0, 2)
    q, s = ops.silu_mul_fp8_quant(x, 0)
    assert q.shape == (2, 0, 128) and s.shape == (2, 0, 1)
    q, s, h = ops.add_rmsnorm_fp8_quant(x, x, torch.ones(256, dtype=torch.float16, device=device), EPS, 128)
    assert q.shape == h.shape == (2, 0, 256)


# ----------------------------------------------------------------------------- together


def _mlp(x, residual, w, group: int = 128):  # type: ignore[no-untyped-def]
    """A decoder's MLP sublayer: residual + norm + codes, gate_up, SiLU * up + codes, down + residual."""
    q, s, h = ops.add_rmsnorm_fp8_quant(x, residual, w["gamma"], EPS, group)
    y = ops.fp8_block_linear(q, s, w["gu"], w["gus"], None, x.dtype, "hip")
    q, s = ops.silu_mul_fp8_quant(y, group)
    return ops.fp8_block_linear(q, s, w["down"], w["downs"], None, x.dtype, "hip", "residual", h)


def _mlp_weights(h: int, inter: int, dtype: torch.dtype, device: torch.device) -> dict[str, torch.Tensor]:
    _, _, gu, gus = bc.linear_inputs(1, 2 * inter, h, seed=5)
    _, _, down, downs = bc.linear_inputs(1, h, inter, seed=6)
    gamma = (1 + 0.1 * torch.randn((h,), generator=bc.gen("gamma", h))).to(dtype)
    out = {"gu": gu, "gus": gus / 64, "down": down, "downs": downs / 64, "gamma": gamma}
    return {name: t.to(device) for name, t in out.items()}


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_mlp_sublayer_and_its_graph(m: int, dtype: torch.dtype, device: torch.device) -> None:
    """The four operators as a decoder's MLP runs them, against the host route's torch expressions (each
    step's codes may differ by a rounding, so the whole agrees as two roundings of the codes do), and
    captured in a graph on a stream of its own, replayed on new inputs with eager work in between."""
    h, inter = 512, 640
    w = _mlp_weights(h, inter, dtype, device)
    inputs = [(bc.rows(m, h, dtype, seed=10 + i).to(device), bc.rows(m, h, dtype, seed=20 + i).to(device))
              for i in range(3)]
    eager = [_mlp(*i, w) for i in inputs]
    for (x, r), y in zip(inputs, eager):
        cpu = {name: t.cpu() for name, t in w.items()}
        want = _mlp(x.cpu(), r.cpu(), cpu).double()
        err = float((y.cpu().double() - want).norm() / want.norm())
        assert err <= 2e-2, err
    x, r = (t.clone() for t in inputs[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            side = _mlp(x, r, w)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(side, eager[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _mlp(x, r, w)
    for i in (1, 2, 0, 1):
        x.copy_(inputs[i][0])
        r.copy_(inputs[i][1])
        graph.replay()
        assert torch.equal(out, eager[i]), i
        assert torch.equal(_mlp(*inputs[2], w), eager[2])
        torch.cuda.synchronize()


def test_opcheck(device: torch.device) -> None:
    # opcheck's schema test does arithmetic on inputs, which torch has no kernel for in float8.
    tests = ("test_faketensor", "test_aot_dispatch_dynamic")
    x = bc.rows(3, 256, torch.float16).to(device)
    w = torch.ones(256, dtype=torch.float16, device=device)
    for group in (128, 0):
        opcheck(ops.fp8_quant.default, (x, group), test_utils=tests)
        opcheck(ops.silu_mul_fp8_quant.default, (x, group), test_utils=tests)
        opcheck(ops.add_rmsnorm_fp8_quant.default, (x, x, w, EPS, group), test_utils=tests)
        opcheck(ops.add_rmsnorm_fp8_quant.default, (x, None, w, EPS, group), test_utils=tests)
    d = _to(device, bc.linear_inputs(3, 130, 272))
    r = torch.zeros((3, 130), dtype=torch.bfloat16, device=device)
    opcheck(ops.fp8_block_linear.default, (*d, None, torch.bfloat16, "hip"), test_utils=tests)
    opcheck(ops.fp8_block_linear.default, (*d, None, torch.bfloat16, "hip", "residual", r), test_utils=tests)


def test_torch_compile_of_the_mlp(device: torch.device) -> None:
    w = _mlp_weights(256, 256, torch.float16, device)
    fn = torch.compile(lambda x, r: _mlp(x, r, w), backend="aot_eager", fullgraph=True, dynamic=True)
    for m in (5, 33):
        x, r = bc.rows(m, 256, torch.float16, 8).to(device), bc.rows(m, 256, torch.float16, 9).to(device)
        assert torch.equal(fn(x, r), _mlp(x, r, w))


def test_gpu_calls_refuse_host_tensors(device: torch.device) -> None:
    x8, xs, w8, ws = _to(device, bc.linear_inputs(2, 16, 128))
    with pytest.raises(ValueError, match="one device"):
        ops.fp8_block_linear(x8, xs, w8.cpu(), ws, None, torch.float16, "hip")
    x = torch.zeros((2, 128), dtype=torch.float16, device=device)
    with pytest.raises(ValueError, match="one device"):
        ops.add_rmsnorm_fp8_quant(x, x.cpu(), torch.ones(128, dtype=torch.float16, device=device), EPS, 128)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.fp8_block_linear(x8[:, :120], xs, w8[:, :120], ws, None, torch.float16, "hip")
