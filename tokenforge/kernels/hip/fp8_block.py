"""FP8 (e4m3fn) with a scale per 128: the quantizers and the block-scaled linear on gfx950.

No counterpart in the reference, whose one quantizer (rmsnorm_fp8.py) writes a scale per row and whose
linears have int4 weights. The quantizers write codes and scales of three producers in one launch each;
``fp8_block_linear`` multiplies such codes with e4m3 weights that have a scale per 128 x 128 block, the
form in which FP8 checkpoints are published.
"""

from __future__ import annotations

import ctypes

import torch

from tokenforge.kernels import _lib
from tokenforge.kernels.block_config import BLOCK, BlockConfig
from tokenforge.kernels.hip._common import on_device, ptr, require_gpu, stream_of

DTYPES = {torch.float16: 0, torch.bfloat16: 1}  # TF_DTYPE_* of the C header
GROUP_SIZES = (BLOCK, 0)
MAX_CODE_STRIDE = 1 << 22  # rows of codes start less than 4 MiB apart, rows of x_scale less than 2^20 elements:
MAX_SCALE_STRIDE = 1 << 20  # a tile's offsets stay in 31 bits (rows further apart are copied)


def blocks(size: int) -> int:
    """Blocks of 128 that cover ``size``."""
    return -(-size // BLOCK)


# ----------------------------------------------------------------------------- quantizers


def check_quant_input(x: torch.Tensor, group_size: int, *, halves: int = 1, whole_row: bool = False) -> tuple[int, int]:
    """Checks of a quantizer's input ``x [T, halves * K]``; returns ``(T, K)``."""
    if x.dim() != 2:
        raise ValueError(f"x must be 2-D [T, K], got {tuple(x.shape)}")
    if x.dtype not in DTYPES:
        raise TypeError(f"x must be fp16 or bf16, got {x.dtype}")
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be {BLOCK}, or 0 for one scale per row, got {group_size}")
    t, width = x.shape
    if width % halves:
        raise ValueError(f"x must hold gate and up halves of one length, got a last dimension of {width}")
    k = width // halves
    if k == 0:
        raise ValueError("x must have a last dimension above 0")
    if (whole_row or group_size == 0) and k > _lib.FP8_MAX_ROW:
        raise ValueError(f"rows above {_lib.FP8_MAX_ROW} are not supported, got {k}")
    return t, k


def check_norm_args(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                    group_size: int) -> tuple[int, int]:
    """Checks of the norm's arguments; returns ``(T, H)``."""
    t, h = check_quant_input(x, group_size, whole_row=True)
    if tuple(weight.shape) != (h,):
        raise ValueError(f"weight shape {tuple(weight.shape)} != {(h,)}")
    if weight.dtype != x.dtype:
        raise TypeError(f"weight must be {x.dtype} like x, got {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be {x.dtype} like x, got {residual.dtype}")
    return t, h


def _outputs(t: int, k: int, group_size: int, dev: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    q = torch.empty((t, k), dtype=torch.float8_e4m3fn, device=dev)
    return q, torch.empty((t, blocks(k) if group_size else 1), dtype=torch.float32, device=dev)


def rows(x: torch.Tensor, limit: int = 1 << 62) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous, do not overlap and start less than ``limit`` elements apart;
    a copy only when needed."""
    if x.stride(1) == 1 and (x.shape[0] <= 1 or x.shape[1] <= x.stride(0) < limit):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _row_stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def fp8_quant(x: torch.Tensor, group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [T, K]`` fp16 or bf16 -> ``(q [T, K] float8_e4m3fn, scale)``: ``scale = max(amax / 448,
    1 / (448 * 512))`` fp32, ``[T, ceil(K / 128)]`` over each 128 of a row (``group_size`` 128) or ``[T,
    1]`` over the row (0)."""
    t, k = check_quant_input(x, group_size)
    dev = require_gpu("fp8_quant", x)
    x = rows(x)
    q, s = _outputs(t, k, group_size, dev)
    if t:
        with on_device(dev):
            rc = _lib.lib().tf_fp8_quant(x.data_ptr(), _row_stride(x), DTYPES[x.dtype], q.data_ptr(), s.data_ptr(), t,
                                         k, group_size, stream_of(dev))
        _lib.check(rc, "tf_fp8_quant")
    return q, s


def silu_mul_fp8_quant(x: torch.Tensor, group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`fp8_quant` of ``silu(x[:, :K]) * x[:, K:]`` for ``x [T, 2K]``, in fp32 up to the codes."""
    t, k = check_quant_input(x, group_size, halves=2)
    dev = require_gpu("silu_mul_fp8_quant", x)
    x = rows(x)
    q, s = _outputs(t, k, group_size, dev)
    if t:
        with on_device(dev):
            rc = _lib.lib().tf_silu_mul_fp8_quant(x.data_ptr(), _row_stride(x), DTYPES[x.dtype], q.data_ptr(),
                                                  s.data_ptr(), t, k, group_size, stream_of(dev))
        _lib.check(rc, "tf_silu_mul_fp8_quant")
    return q, s


def add_rmsnorm_fp8_quant(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, group_size: int
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(q, scale, hidden)``: ``hidden = x + residual`` in x's type, then :func:`fp8_quant` of its RMSNorm
    ``hidden / sqrt(mean(hidden^2) + eps) * weight``, in fp32 up to the codes. Without a residual the norm
    is x's and ``hidden`` an empty tensor."""
    t, h = check_norm_args(x, residual, weight, group_size)
    dev = require_gpu("add_rmsnorm_fp8_quant", *(a for a in (x, residual, weight) if a is not None))
    x, weight = rows(x), weight.contiguous()
    residual = None if residual is None else rows(residual)
    q, s = _outputs(t, h, group_size, dev)
    hidden = torch.empty((t, h) if residual is not None else (0,), dtype=x.dtype, device=dev)
    if t:
        with on_device(dev):
            rc = _lib.lib().tf_add_rmsnorm_fp8_quant(
                x.data_ptr(), _row_stride(x), ptr(residual), 0 if residual is None else _row_stride(residual),
                weight.data_ptr(), DTYPES[x.dtype], q.data_ptr(), s.data_ptr(),
                None if residual is None else hidden.data_ptr(), t, h, float(eps), group_size, stream_of(dev))
        _lib.check(rc, "tf_add_rmsnorm_fp8_quant")
    return q, s, hidden


# ----------------------------------------------------------------------------- linear


def check_block_linear(
    x8: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    w_scale: torch.Tensor,
    bias: torch.Tensor | None,
    out_dtype: torch.dtype,
    residual: torch.Tensor | None,
) -> tuple[int, int, int]:
    """Every check of the block-scaled linear, on any device; returns ``(M, N, K)``."""
    if out_dtype not in DTYPES:
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    if x8.dim() != 2 or weight.dim() != 2:
        raise ValueError(f"x8 must be 2-D [M, K] and weight 2-D [N, K], got {tuple(x8.shape)} and {tuple(weight.shape)}")
    if x8.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise TypeError(f"x8 and weight must be float8_e4m3fn, got {x8.dtype} and {weight.dtype}")
    m, k = x8.shape
    n = weight.shape[0]
    if weight.shape[1] != k:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match K={k}")
    if k == 0 or k % 16 or k >= MAX_CODE_STRIDE:
        raise ValueError(f"K must be a multiple of 16 below {MAX_CODE_STRIDE}, got {k}")
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError(f"x_scale and w_scale must be fp32, got {x_scale.dtype} and {w_scale.dtype}")
    if tuple(x_scale.shape) != (m, blocks(k)):
        raise ValueError(f"x_scale shape {tuple(x_scale.shape)} != {(m, blocks(k))}")
    if tuple(w_scale.shape) != (blocks(n), blocks(k)):
        raise ValueError(f"w_scale shape {tuple(w_scale.shape)} != {(blocks(n), blocks(k))}")
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)} != {(n,)}")
        if bias.dtype != out_dtype:
            raise TypeError(f"bias must be {out_dtype} like the output, got {bias.dtype}")
    if residual is not None:
        if tuple(residual.shape) != (m, n):
            raise ValueError(f"residual shape {tuple(residual.shape)} != {(m, n)}")
        if residual.dtype != out_dtype:
            raise TypeError(f"residual must be {out_dtype} like the output, got {residual.dtype}")
    return m, n, k


def _code_rows(t: torch.Tensor) -> torch.Tensor:
    """:func:`rows` that start on 16 bytes (the kernels use 128-bit loads)."""
    t = rows(t, MAX_CODE_STRIDE)
    if t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.stride(0) % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def to_c_config(cfg: BlockConfig) -> _lib.TfGemmConfig:
    return _lib.TfGemmConfig(_lib.BLOCK_KERNEL_IDS[cfg.kernel], cfg.block_m, cfg.block_n, BLOCK, cfg.split_k,
                             cfg.num_warps, cfg.num_stages)


def workspace_bytes(m: int, n: int, k: int, cfg: BlockConfig) -> int:
    c = to_c_config(cfg)
    need = int(_lib.lib().tf_fp8_block_workspace_bytes(m, n, k, ctypes.byref(c)))
    if need < 0:
        raise ValueError(f"{cfg} is not a compiled config")
    return need


def fp8_block_gemm(
    x8: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    w_scale: torch.Tensor,
    config: BlockConfig,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float16,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x8 [M, K]`` x ``weight [N, K]`` -> ``[M, N]`` with the launch ``config`` (``tf_fp8_block_linear``)."""
    m, n, k = check_block_linear(x8, x_scale, weight, w_scale, bias, out_dtype, residual)
    dev = require_gpu("fp8_block_linear", *(t for t in (x8, x_scale, weight, w_scale, bias, residual) if t is not None))
    out = torch.empty((m, n), dtype=out_dtype, device=dev)
    if m == 0 or n == 0:
        return out
    x8, weight = _code_rows(x8), _code_rows(weight)
    x_scale, w_scale = rows(x_scale, MAX_SCALE_STRIDE), rows(w_scale)
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else rows(residual)
    c = to_c_config(config)
    need = workspace_bytes(m, n, k, config)
    ws = torch.empty((need + 3) // 4, dtype=torch.float32, device=dev) if need else None
    with on_device(dev):
        rc = _lib.lib().tf_fp8_block_linear(
            x8.data_ptr(), _row_stride(x8), x_scale.data_ptr(), _row_stride(x_scale), weight.data_ptr(),
            _row_stride(weight), w_scale.data_ptr(), _row_stride(w_scale), ptr(bias), ptr(residual),
            0 if residual is None else _row_stride(residual), out.data_ptr(), n, DTYPES[out_dtype], m, n, k,
            ctypes.byref(c), ptr(ws), need, stream_of(dev))
    _lib.check(rc, "tf_fp8_block_linear")
    return out
