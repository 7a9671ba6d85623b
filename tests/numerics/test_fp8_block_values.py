"""FP8 with a scale per 128 on the GPU, further values: gates whose sigmoid leaves fp32's normal range."""

from __future__ import annotations

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import block_codes

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge


@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("k", [128, 130, 1000, 4864])
def test_silu_mul_of_gates_far_below_zero(k: int, group: int, device: torch.device) -> None:
    x = block_codes.far_gates(k)
    block_codes.check_far_gates(*ops.silu_mul_fp8_quant(x.to(device), group), x, group)
