"""FP8 with a scale per 128, the parts that need no GPU: the host route against the definitions in 64
bits, refusals of the operators and of the C entry points, fakes, and the launch rule."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401
from oracle import fp8_block as oblk
from tests.numerics import block_cases as bc
from tests.numerics import block_codes
from tokenforge.kernels import _lib
from tokenforge.kernels.block_config import BLOCK_TILES, block_config
from tokenforge.kernels.hip import fp8_block
from tokenforge.kernels.metrics import KERNEL_CALLS

ops = torch.ops.tokenforge
EPS = 1e-6
F8 = torch.float8_e4m3fn


# ----------------------------------------------------------------------------- host route


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize(("t", "k"), [(1, 128), (3, 130), (2, 7), (5, 1296)])
def test_host_quantizers(t: int, k: int, group: int, dtype: torch.dtype) -> None:
    x, r = bc.rows(t, k, dtype), bc.rows(t, k, dtype, seed=1)
    q, s = ops.fp8_quant(x, group)
    bc.check_codes(q, s, x.double().numpy(), 0.0, group, "fp8_quant")
    gu = bc.rows(t, 2 * k, dtype, seed=2)
    q, s = ops.silu_mul_fp8_quant(gu, group)
    err = (8 + 2 * np.abs(gu.double().numpy()[:, :k])) * bc.U32
    bc.check_codes(q, s, oblk.silu_mul(gu.double().numpy()), err, group, "silu_mul_fp8_quant")
    w = (torch.rand((k,), generator=bc.gen("w", k)) + 0.5).to(dtype)
    q, s, hidden = ops.add_rmsnorm_fp8_quant(x, r, w, EPS, group)
    assert torch.equal(hidden, x + r)
    # torch's mean adds up to k squares in an order of its own: k / 2 roundings of the mean at most.
    y = oblk.rmsnorm((x + r).double().numpy(), w.double().numpy(), EPS)
    bc.check_codes(q, s, y, (k / 2 + 8) * bc.U32, group, "norm")
    assert ops.add_rmsnorm_fp8_quant(x, None, w, EPS, group)[2].shape == (0,)


@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("k", [128, 130])
def test_host_silu_mul_of_gates_far_below_zero(k: int, group: int) -> None:
    x = block_codes.far_gates(k)
    block_codes.check_far_gates(*ops.silu_mul_fp8_quant(x, group), x, group)


@pytest.mark.parametrize("dtype", bc.DTYPES, ids=str)
@pytest.mark.parametrize(("m", "n", "k"), [(1, 1, 16), (3, 130, 144), (2, 300, 1296)])
def test_host_linear(m: int, n: int, k: int, dtype: torch.dtype) -> None:
    inputs = bc.linear_inputs(m, n, k)
    g = bc.gen("extras", m, n)
    bias, res = torch.randn((n,), generator=g).to(dtype), torch.randn((m, n), generator=g).to(dtype)
    KERNEL_CALLS.reset()
    x8, xs, w8, ws = inputs
    y, size, length = oblk.linear(bc.codes(x8), xs.numpy(), bc.codes(w8), ws.numpy())
    for extra in (bias.double().numpy(), res.double().numpy()):
        y, size = y + extra, size + np.abs(extra)
    got = ops.fp8_block_linear(*inputs, bias, dtype, "hip", "residual", res).double().numpy()
    # the host rounds each dequantized operand to fp32 and adds k products in an order of its own
    over = np.abs(got - y) - bc.linear_bound(y, size, length, k, dtype) - (k + 4) * 2 * bc.U32 * size
    assert over.max() <= 0
    assert KERNEL_CALLS.value(kernel="torch_reference", bucket=str({1: 1, 3: 4, 2: 2}[m])) == 1


def test_leading_dimensions_and_empty_rows() -> None:
    x = bc.rows(6, 200, torch.bfloat16).reshape(2, 3, 200)
    q, s = ops.fp8_quant(x, 128)
    assert q.shape == (2, 3, 200) and s.shape == (2, 3, 2) and q.dtype == F8
    assert ops.silu_mul_fp8_quant(x, 0)[1].shape == (2, 3, 1)
    x8, xs, w8, ws = bc.linear_inputs(6, 40, 144)
    y = ops.fp8_block_linear(x8.reshape(2, 3, 144), xs.reshape(2, 3, 2), w8, ws, None, torch.float16, "hip")
    assert y.shape == (2, 3, 40)
    y = ops.fp8_block_linear(x8[:0], xs[:0], w8, ws, None, torch.float16, "hip")
    assert y.shape == (0, 40)
    y = ops.fp8_block_linear(x8, xs, w8[:0], ws[:0], None, torch.float16, "hip")
    assert y.shape == (6, 0)


# ----------------------------------------------------------------------------- refusals


def test_quantizers_refuse() -> None:
    x = torch.zeros((2, 256), dtype=torch.float16)
    w = torch.ones(256, dtype=torch.float16)
    for op in (ops.fp8_quant, ops.silu_mul_fp8_quant):
        with pytest.raises(TypeError, match="fp16 or bf16"):
            op(x.float(), 128)
        with pytest.raises(ValueError, match="group_size"):
            op(x, 64)
        with pytest.raises(ValueError, match="above 0"):
            op(x[:, :0], 128)
        with pytest.raises(ValueError, match="32768"):
            op(torch.zeros((1, 2 * 32769), dtype=torch.float16), 0)
    with pytest.raises(ValueError, match="halves"):
        ops.silu_mul_fp8_quant(x[:, :255], 128)
    with pytest.raises(ValueError, match="weight shape"):
        ops.add_rmsnorm_fp8_quant(x, None, w[:255], EPS, 128)
    with pytest.raises(TypeError, match="weight must be"):
        ops.add_rmsnorm_fp8_quant(x, None, w.float(), EPS, 128)
    with pytest.raises(ValueError, match="residual shape"):
        ops.add_rmsnorm_fp8_quant(x, x[:1], w, EPS, 128)
    with pytest.raises(TypeError, match="residual must be"):
        ops.add_rmsnorm_fp8_quant(x, x.bfloat16(), w, EPS, 128)
    with pytest.raises(ValueError, match="32768"):
        ops.add_rmsnorm_fp8_quant(torch.zeros((1, 32769), dtype=torch.float16), None,
                                  torch.ones(32769, dtype=torch.float16), EPS, 128)


def test_linear_refuses() -> None:
    x8, xs, w8, ws = bc.linear_inputs(2, 130, 256)
    bias, res = torch.zeros(130, dtype=torch.float16), torch.zeros((2, 130), dtype=torch.float16)

    def call(x8=x8, xs=xs, w8=w8, ws=ws, bias=None, dtype=torch.float16, backend="hip", epilogue="none",  # type: ignore[no-untyped-def]
             residual=None):
        return ops.fp8_block_linear(x8, xs, w8, ws, bias, dtype, backend, epilogue, residual)

    call()
    cases = [
        (ValueError, "op level", {"backend": "marlin"}),
        (ValueError, "epilogue must be", {"epilogue": "silu_mul"}),
        (ValueError, "goes with epilogue", {"residual": res}),
        (ValueError, "goes with epilogue", {"epilogue": "residual"}),
        (ValueError, "residual shape", {"epilogue": "residual", "residual": res[:1]}),
        (TypeError, "residual must be", {"epilogue": "residual", "residual": res.float()}),
        (TypeError, "out_dtype", {"dtype": torch.float32}),
        (TypeError, "float8_e4m3fn", {"x8": x8.float()}),
        (TypeError, "float8_e4m3fn", {"w8": w8.view(torch.uint8)}),
        (ValueError, "does not match K", {"w8": w8[:, :128]}),
        (ValueError, "multiple of 16", {"x8": x8[:, :250], "w8": w8[:, :250]}),
        (TypeError, "fp32", {"xs": xs.half()}),
        (TypeError, "fp32", {"ws": ws.double()}),
        (ValueError, "x_scale shape", {"xs": xs[:, :1]}),
        (ValueError, "x_scale shape", {"xs": xs[:1]}),
        (ValueError, "w_scale shape", {"ws": ws[:1]}),
        (ValueError, "bias shape", {"bias": bias[:129]}),
        (TypeError, "bias must be", {"bias": bias.bfloat16()}),
        (ValueError, "weight", {"w8": w8[0]}),
        (ValueError, "below", {"x8": torch.zeros((1, 1 << 22), dtype=torch.uint8).view(F8), "xs": xs[:1],
                               "w8": torch.zeros((1, 1 << 22), dtype=torch.uint8).view(F8)}),
    ]
    for error, match, args in cases:
        with pytest.raises(error, match=match):
            call(**args)


# Fake device addresses: 16-byte aligned, never dereferenced (every call is refused on the host).
_X, _S, _W, _T, _O, _WS = (0x10000 * (i + 1) for i in range(6))


def _entry(m: int = 4, n: int = 64, k: int = 256, cfg: tuple[int, ...] = (4, 16, 16, 128, 1, 4, 4), dtype: int = 0,
           x: int = _X, ldx: int = 256, ldxs: int = 2, ldw: int = 256, ldws: int = 2, ldo: int = 64, ldr: int = 64,
           residual: int | None = None, ws: int | None = None, ws_bytes: int = 0) -> tuple[int, bytes]:
    h = _lib.lib()
    c = _lib.TfGemmConfig(*cfg)
    rc = h.tf_fp8_block_linear(x, ldx, _S, ldxs, _W, ldw, _T, ldws, None, residual, ldr, _O, ldo, dtype, m, n, k,
                               ctypes.byref(c), ws, ws_bytes, None)
    return rc, h.tf_last_error()


@pytest.mark.parametrize(("args", "message"), [
    ({"dtype": 2}, b"dtype"), ({"k": 250}, b"multiple of 16"), ({"k": 0}, b"bad size"), ({"m": -1}, b"bad size"),
    ({"m": 1 << 31}, b"bad size"), ({"ldx": 240}, b"row stride"), ({"ldxs": 1}, b"row stride"),
    ({"ldo": 63}, b"row stride"), ({"residual": _O, "ldr": 1}, b"row stride"), ({"ldx": 264}, b"16-byte"),
    ({"x": _X + 8}, b"16-byte"), ({"ldw": 264}, b"16-byte"), ({"cfg": (1, 16, 16, 128, 1, 8, 1)}, b"compiled config"),
    ({"cfg": (4, 48, 16, 128, 1, 8, 1)}, b"compiled"), ({"x": 0}, b"null pointer"),
    ({"cfg": (5, 256, 256, 64, 1, 8, 2)}, b"compiled"), ({"cfg": (5, 256, 256, 128, 0, 8, 2)}, b"compiled"),
    ({"cfg": (5, 32, 64, 128, 1, 8, 3), "m": (1 << 31) - 1, "k": 16, "n": 64}, b"too many tiles"),
    ({"cfg": (5, 64, 64, 128, 2, 8, 4)}, b"workspace too small"),
    ({"cfg": (5, 64, 64, 128, 2, 8, 4), "ws": _WS + 8, "ws_bytes": 1 << 20}, b"16-byte"),
    ({"k": 1 << 22, "ldx": 1 << 22, "ldw": 1 << 22, "ldxs": 1 << 15, "ldws": 1 << 15}, b"apart"),
    ({"ldxs": 1 << 20}, b"apart"),
])
def test_linear_entry_refuses_on_the_host(args: dict, message: bytes) -> None:  # type: ignore[type-arg]
    rc, text = _entry(**args)
    assert rc == _lib.TF_EINVAL and message in text, text


def test_quantizer_entries_refuse_on_the_host() -> None:
    h = _lib.lib()
    cases = [
        (h.tf_fp8_quant(_X, 128, 2, _O, _S, 4, 128, 128, None), b"dtype"),
        (h.tf_fp8_quant(_X, 128, 0, _O, _S, 4, 128, 64, None), b"group_size"),
        (h.tf_fp8_quant(_X, 127, 0, _O, _S, 4, 128, 128, None), b"row stride"),
        (h.tf_fp8_quant(None, 128, 0, _O, _S, 4, 128, 128, None), b"null"),
        (h.tf_fp8_quant(_X, 40000, 0, _O, _S, 4, 40000, 0, None), b"32768"),
        (h.tf_fp8_quant(_X, 1 << 40, 0, _O, _S, 4, 1 << 40, 128, None), b"too long"),
        (h.tf_fp8_quant(_X, 128, 0, _O, _S, 1 << 31, 128, 128, None), b"too many"),
        (h.tf_silu_mul_fp8_quant(_X, 255, 0, _O, _S, 4, 128, 128, None), b"row stride"),
        (h.tf_silu_mul_fp8_quant(_X, 256, 0, _O, _S, 4, 0, 128, None), b"k > 0"),
        (h.tf_add_rmsnorm_fp8_quant(_X, 128, None, 0, None, 0, _O, _S, None, 4, 128, EPS, 128, None), b"null"),
        (h.tf_add_rmsnorm_fp8_quant(_X, 128, _X, 128, _W, 0, _O, _S, None, 4, 128, EPS, 128, None), b"null"),
        (h.tf_add_rmsnorm_fp8_quant(_X, 128, _X, 64, _W, 0, _O, _S, _T, 4, 128, EPS, 128, None), b"row stride"),
        (h.tf_add_rmsnorm_fp8_quant(_X, 40000, None, 0, _W, 0, _O, _S, None, 4, 40000, EPS, 128, None), b"32768"),
    ]
    assert all(rc == _lib.TF_EINVAL for rc, _ in cases)
    # (each call's own message: the last one stays)
    assert b"32768" in h.tf_last_error()
    assert h.tf_fp8_quant(_X, 128, 0, _O, _S, 0, 128, 128, None) == _lib.TF_OK  # no rows, no launch


@pytest.mark.parametrize("k", [0, -1, 5 - (1 << 32), -(1 << 62)])
def test_quantizer_entries_refuse_lengths_below_one(k: int) -> None:
    """Negative lengths whose low 32 bits are a positive number too (no rows: nothing is launched either way)."""
    h = _lib.lib()
    for rc in (h.tf_fp8_quant(_X, 128, 0, _O, _S, 0, k, 128, None),
               h.tf_silu_mul_fp8_quant(_X, 256, 0, _O, _S, 0, k, 128, None),
               h.tf_add_rmsnorm_fp8_quant(_X, 128, None, 0, _W, 0, _O, _S, None, 0, k, EPS, 128, None)):
        assert rc == _lib.TF_EINVAL and b"k > 0" in h.tf_last_error()


def test_workspace_bytes_never_wrap() -> None:
    """The partial sums' bytes, or -1 where they pass 63 bits or a size is one the linear refuses."""
    top = (1 << 31) - 1
    for split in (1, 2, 5, 16):
        cfg = ctypes.byref(_lib.TfGemmConfig(5, 64, 64, 128, split, 8, 4))
        for m in (0, 1, 1000, 1 << 28, 1 << 30, top, top + 1, 1 << 40, -1):
            for n in (0, 1, 1000, 1 << 30, 0x7FFFFF00, 0x7FFFFF01, 1 << 40, -1):
                for k in (16, 4096, 0x7FFFFF00, (1 << 63) - 1):
                    got = _lib.lib().tf_fp8_block_workspace_bytes(m, n, k, cfg)
                    bytes_ = 4 * m * n * min(split, -(-k // 128)) if min(split, -(-k // 128)) > 1 else 0
                    known = 0 <= m <= top and 0 <= n <= 0x7FFFFF00 and k <= 0x7FFFFF00 and bytes_ < 1 << 63
                    assert got == (bytes_ if known else -1), (m, n, k, split)


# ----------------------------------------------------------------------------- fakes and the launch rule


def test_fake_tensor_shapes() -> None:
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        f = mode.from_tensor
        x = f(torch.zeros((2, 3, 300), dtype=torch.bfloat16))
        q, s = ops.fp8_quant(x, 128)
        assert q.shape == (2, 3, 300) and q.dtype == F8 and s.shape == (2, 3, 3) and s.dtype == torch.float32
        q, s = ops.silu_mul_fp8_quant(x, 0)
        assert q.shape == (2, 3, 150) and s.shape == (2, 3, 1)
        w = f(torch.ones(300, dtype=torch.bfloat16))
        q, s, h = ops.add_rmsnorm_fp8_quant(x, x, w, EPS, 128)
        assert h.shape == x.shape and h.dtype == x.dtype
        assert ops.add_rmsnorm_fp8_quant(x, None, w, EPS, 128)[2].shape == (0,)
        x8, xs, w8, ws = (f(t) for t in bc.linear_inputs(6, 40, 144))
        y = ops.fp8_block_linear(x8.reshape(2, 3, 144), xs.reshape(2, 3, 2), w8, ws, None, torch.bfloat16, "hip")
        assert y.shape == (2, 3, 40) and y.dtype == torch.bfloat16


def test_the_rule_names_compiled_configs() -> None:
    for m in (1, 2, 8, 16, 17, 33, 64, 65, 128, 129, 200, 333, 512, 1000, 2048, 4096, 100000):
        for n, k in ((1, 16), (64, 128), (896, 896), (1000, 1296), (4608, 3584), (3584, 18944), (37888, 3584)):
            cfg = block_config(m, n, k)
            assert (cfg.kernel, cfg.block_m, cfg.block_n, cfg.num_warps, cfg.num_stages) in BLOCK_TILES
            assert 1 <= cfg.split_k <= max(1, -(-k // 128))
            assert fp8_block.workspace_bytes(m, n, k, cfg) >= 0


def test_the_rule_stays_within_one_launch() -> None:
    """Every call that some compiled config can launch (fewer than 2^32 threads) gets one that can."""
    for m, n, k in ((1, 300_000_000, 16), (4, 300_000_000, 16), (2, 150_000_000, 2048), (16, 300_000_000, 16),
                    (300, 140_000_000, 16), (1, 0x7FFFFF00, 16), (1 << 30, 1, 16), ((1 << 30) + 5, 1, 16),
                    (280_000_000, 16, 16), (0x7FFFFF00, 1, 16)):
        c = block_config(m, n, k)
        gemv = c.kernel == "gemv_block"  # rows on the grid's second axis
        groups = (1 if gemv else -(-m // c.block_m)) * -(-n // c.block_n) * c.split_k
        assert groups * 64 * c.num_warps < 1 << 32, (m, n, k, c)


# ----------------------------------------------------------------------------- the oracle


def test_oracle_linear_against_scalar_loops() -> None:
    from fractions import Fraction

    from oracle.reference import e4m3_decode

    x8, xs, w8, ws = bc.linear_inputs(2, 130, 144)
    y, size, length = oblk.linear(bc.codes(x8), xs.numpy(), bc.codes(w8), ws.numpy())
    xd, wd = e4m3_decode(bc.codes(x8)), e4m3_decode(bc.codes(w8))
    for m, n in ((0, 0), (1, 127), (1, 129)):
        terms = [Fraction(float(xd[m, k])) * Fraction(float(wd[n, k])) * Fraction(float(xs[m, k // 128]))
                 * Fraction(float(ws[n // 128, k // 128])) for k in range(144)]
        assert abs(float(sum(terms)) - y[m, n]) <= 144 * 2.0**-52 * size[m, n]
        assert abs(float(sum(abs(t) for t in terms)) - size[m, n]) <= 144 * 2.0**-52 * size[m, n]
        assert abs(float(sum(t * t for t in terms)) ** 0.5 - length[m, n]) <= 144 * 2.0**-52 * length[m, n]


@pytest.mark.parametrize("group", [128, 0])
def test_code_check_refuses_wrong_codes_and_scales(group: int) -> None:
    """The check itself: right codes pass; a NaN code, a code one step off, a sign and a wrong scale do not."""
    x = bc.rows(5, 260, torch.float16, seed=40)
    y = x.double().numpy()
    q, s = ops.fp8_quant(x, group)
    block_codes.check_codes(q, s, y, 0.0, group, "right")
    at = [int(i) for i in np.unravel_index(np.abs(bc.codes(q) & 0x7F).argmax(), q.shape)]

    def planted(code: int) -> torch.Tensor:
        out = q.view(torch.uint8).clone()
        out[at[0], at[1]] = code
        return out.view(F8)

    right = int(bc.codes(q)[at[0], at[1]])
    for code in (0x7F, 0xFF, right - 1, right ^ 0x80, 0):
        with pytest.raises(AssertionError):
            block_codes.check_codes(planted(code), s, y, 0.0, group, "planted")
    with pytest.raises(AssertionError):  # every code
        block_codes.check_codes(torch.full(q.shape, 0x7F, dtype=torch.uint8).view(F8), s, y, 0.0, group, "planted")
    for wrong in (float("nan"), float("inf"), 0.0, float(s[at[0], 0]) * (1 + 2.0**-20)):
        t = s.clone()
        t[at[0], 0] = wrong
        with pytest.raises(AssertionError):
            block_codes.check_codes(q, t, y, 0.0, group, "planted")


@pytest.mark.parametrize("kind", ["outliers", "one sign", "cancelling"])
def test_remainder_check_against_the_stated_rule(kind: str) -> None:
    """The check of the linear's remainder: the rule itself (products cut toward zero in groups of eight) passes,
    a cut four bits higher, a group left out and a NaN do not."""
    from oracle.reference import e4m3_decode

    inputs = block_codes.hard_inputs(kind, 3, 10, 272)
    residual = block_codes.remainder_residual(inputs)
    x8, xs, w8, ws = inputs
    p = e4m3_decode(bc.codes(x8)).astype(np.float64)[:, None] * e4m3_decode(bc.codes(w8)).astype(np.float64)[None]
    scale = xs.double().numpy()[:, None] * np.repeat(ws.double().numpy(), 128, axis=0)[:10][None]

    def linear(bits: int, skip: int = -1) -> torch.Tensor:
        y = np.zeros(p.shape[:2])
        for g, k0 in enumerate(range(0, 272, 8)):
            part = p[:, :, k0:k0 + 8]
            unit = np.exp2(np.floor(np.log2(np.abs(part).max(axis=2, keepdims=True))) - bits)
            y += 0.0 if g == skip else (np.trunc(part / unit) * unit).sum(axis=2) * scale[:, :, k0 // 128]
        return torch.from_numpy(y + residual.double().numpy()).to(torch.float16)

    block_codes.check_remainder(linear(13), inputs, residual, "the rule")
    block_codes.check_remainder(linear(40), inputs, residual, "no cut")
    nan = linear(13)
    nan[1, 2] = float("nan")
    # ("cancelling": by the rule a group's sum is lost whole)
    for wrong in (nan,) if kind == "cancelling" else (linear(9), linear(13, 5), nan):
        with pytest.raises(AssertionError):
            block_codes.check_remainder(wrong, inputs, residual, "planted")


def test_oracle_half_step_and_scales() -> None:
    values = np.sort(np.unique(np.abs(torch.arange(0, 127, dtype=torch.uint8).view(F8).float().numpy()))).astype(np.float64)
    for lo, hi in zip(values[:-1], values[1:]):
        assert oblk.half_step(np.array([lo]))[0] == (hi - lo) / 2, lo
    y = np.array([[1.0, -448.0] + [0.0] * 126 + [-896.0, 2.0]])
    assert np.array_equal(oblk.block_scales(y, 128), [[1.0, 2.0]])
    assert np.array_equal(oblk.block_scales(y, 0), [[2.0]])
    assert np.array_equal(oblk.block_scales(np.zeros((1, 3)), 128), [[1.0 / (448 * 512)]])
    assert np.array_equal(oblk.spread(np.array([[1.0, 2.0]]), 130, 128), [[1.0] * 128 + [2.0] * 2])
