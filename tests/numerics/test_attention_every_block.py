"""Large calls of the paged attention, every output of them: the same sequences again and again, wherever their items begin
and end among the workgroups. Bound: ``kv_cases.check_attention``'s, computed once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from oracle import kv_cache as okv
from tests.numerics import kv_cases as kc

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]
LINE = 1 << 15


def _queries(m: int, q_heads: int, d: int, dtype: torch.dtype) -> torch.Tensor:
    q = torch.randn((m, q_heads, d), generator=kc.gen("q", m, q_heads, d, "every block"))
    q[..., :: max(1, d // 4)] *= 2.0
    return q.to(dtype)


def _want(q: torch.Tensor, c: kc.Cache, table: torch.Tensor, lens: list[int], scale: float,
          window: int) -> tuple[np.ndarray, np.ndarray]:
    """The outputs in 64 bits and the bound of each, as ``kv_cases.check_attention`` derives it."""
    d, out, bounds = q.shape[2], [], []
    kc64, vc64 = kc.values(c.k.float()), kc.values(c.v.float())
    ks, vs = (None if s is None else kc.values(s) for s in (c.ks, c.vs))
    for b, n in enumerate(lens):
        begin, row = max(0, n - window) if window else 0, table[b].numpy()
        k, v = okv.tokens(kc64, ks, row, begin, n), okv.tokens(vc64, vs, row, begin, n)
        want, size, spread = okv.attention(kc.values(q[b]), k, v, scale)
        e = (d + 16) * kc.MFMA * spread[:, None] + 2.0**-22
        bound = (2 * e + 2.0**-16 + 2 * (k.shape[0] + 64) * kc.MFMA) * size
        bounds.append(bound + kc.EPS[q.dtype] * (np.abs(want) + bound) + (2.0**-25 if q.dtype == torch.float16 else 0.0))
        out.append(want)
    return np.stack(out), np.stack(bounds)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize(("d", "group", "page"), [(64, 4, 16), (64, 20, 16), (128, 7, 16), (128, 20, 16), (256, 4, 16), (96, 4, 16),
                                                  (128, 7, 24), (128, 20, 24), (256, 4, 24)])
@pytest.mark.parametrize("form", ["shared", "whole", "window"])
def test_every_output(form: str, d: int, group: int, page: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    row = 2 * d * (1 if fp8 else 2)
    dp = 64 if d <= 64 else 128 if d <= 128 else 256
    capacity = (512 << 10) // (2 * dp * (1 if fp8 else 2)) // page * page if form == "whole" else LINE
    lens = [min(2049, capacity), capacity // 2 + 1 if form == "whole" else 1777, 1, 0, 300]
    window = 1500 if form == "window" else 0
    table, pages = kc.tables(lens, page, capacity // page)
    c = kc.cache(pages, 2, page, d, dtype, fp8)
    q = _queries(len(lens), 2 * group, d, dtype)
    want, bound = _want(q, c, table, lens, d**-0.5, window)
    cache = c.to(device)
    past = 101 if form == "whole" else (60 << 20) // (sum(lens) * row) + 1  # past the sizes of nontemporal loads
    for n in (past // 5, past):
        out = ops.paged_attention(q.repeat(n, 1, 1).to(device), *cache, table.repeat(n, 1).to(device),
                                  torch.tensor(lens * n, dtype=torch.int32, device=device), d**-0.5, window)
        got = kc.values(out).reshape(n, *want.shape)
        assert np.isfinite(got).all()
        over = (np.abs(got - want) - bound).reshape(n, len(lens), -1).max(-1)
        assert over.max() <= 0, f"block, sequence {np.unravel_index(over.argmax(), over.shape)} of {n}: {over.max():.3e} over"
