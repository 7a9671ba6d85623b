"""The paged attention where the value of the token with the largest score is nothing beside the others': what is left of
the result are probabilities far below it.

Bound. Each score is one product that is not zero, so its sum is exact: the scale times log2(e), the product with it and an
e4m3 scale are 3 roundings of it, the subtraction of the maximum 1 of at most twice it, 5 U32 |score|; the exponential's own
error is within 2^-22. Numerator and denominator have it alike: twice. Sums and joins of n terms: n + 64 additions within
MFMA each, both of them. Probabilities enter the second product as two halves, within 2^-16 of themselves; with 16-bit fp16
values two halves on fp16's subnormal step, the largest as 2^15: within 2^-25 2^-15 = 2^-40 of the largest, which
sum |v| / l of it reaches the result (l: the sum of the probabilities over the largest). Then half a step of the result.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from oracle import kv_cache as okv
from tests.numerics import kv_cases as kc

ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]
D, PAGE, HEADS, GROUP = 64, 16, 2, 3


def _cache(pages: int, table: torch.Tensor, scores: torch.Tensor, values: torch.Tensor, dtype: torch.dtype,
           fp8: bool) -> kc.Cache:
    """Tokens whose keys hold ``scores`` in their first channel and nothing else, and their ``values [n, HEADS, D]``."""
    at, off = table[0, torch.arange(len(scores)) // PAGE].long(), torch.arange(len(scores)) % PAGE
    k, v = (torch.zeros((pages, HEADS, PAGE, D)) for _ in "kv")
    k[at, :, off, 0] = scores[:, None].expand(-1, HEADS)
    v[at, :, off] = values
    out = []
    for x in (k, v):
        if fp8:
            s = (x.abs().amax(-1) / 448.0).clamp(min=1 / (448.0 * 512.0))
            out.append(((x / s[..., None]).clamp(-448, 448).to(kc.F8), s))
        else:
            out.append((x.to(dtype), None))
    (k, ks), (v, vs) = out
    return kc.Cache(k, v, ks, vs)


def _check(out: torch.Tensor, q: torch.Tensor, c: kc.Cache, table: torch.Tensor, n: int, fp8: bool) -> None:
    kv = [okv.tokens(kc.values(x.float()), None if s is None else kc.values(s), table[0].numpy(), 0, n)
          for x, s in ((c.k, c.ks), (c.v, c.vs))]
    want, size, spread = okv.attention(kc.values(q[0]), *kv, 1.0)
    score = np.repeat(kv[0][..., 0], GROUP, 1).T  # [q heads, n]: q is one in the first channel
    ell = np.exp(score - score.max(1, keepdims=True)).sum(1)
    e = 5 * kc.U32 * spread[:, None] + 2.0**-22
    bound = (2 * e + 2.0**-16 + 2 * (n + 64) * kc.MFMA) * size
    if q.dtype == torch.float16 and not fp8:
        bound += 2.0**-40 * np.repeat(np.abs(kv[1]).sum(0), GROUP, 0) / ell[:, None]
    bound += kc.EPS[q.dtype] * (np.abs(want) + bound) + (2.0**-25 if q.dtype == torch.float16 else 0.0)
    over = np.abs(kc.values(out[0]) - want) - bound
    assert over.max() <= 0, f"{over.max():.3e} over the bound, {(np.abs(kc.values(out[0]) / want - 1)).max():.2e} of the result"


def _call(device: torch.device, n: int, gap: float, leader: int, dtype: torch.dtype, fp8: bool, width: int,
          inf: int | None = None) -> tuple[torch.Tensor, torch.Tensor, kc.Cache, torch.Tensor]:
    table, pages = kc.tables([n], PAGE, width)
    scores = -(torch.arange(n) % 7) / 8.0
    scores[leader] = gap
    values = 3e4 + 3e4 * torch.rand((n, HEADS, D), generator=kc.gen("far scores", n))
    values[leader] = 0.0
    if inf is not None:
        values[inf, 0, 5] = float("inf")
    c = _cache(pages, table, scores, values, dtype, fp8)
    q = torch.zeros((1, HEADS * GROUP, D), dtype=dtype)
    q[..., 0] = 1.0
    out = ops.paged_attention(q.to(device), *c.to(device), table.to(device),
                              torch.tensor([n], dtype=torch.int32, device=device), 1.0, 0)
    return out, q, c, table


@pytest.mark.gpu
@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [8.0, 12.0, 17.0, 20.0, 22.0])
@pytest.mark.parametrize(("n", "leader"), [(31, 0), (31, 30), (900, 0), (900, 450), (900, 899)])
@pytest.mark.parametrize("width", [0, 2048], ids=["whole", "shared"])
def test_probabilities_far_below_the_largest(width: int, n: int, leader: int, gap: float, dtype: torch.dtype, fp8: bool,
                                             device: torch.device) -> None:
    out, q, c, table = _call(device, n, gap, leader, dtype, fp8, width)
    _check(out, q, c, table, n, fp8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("gap", [0.0, 12.0, 22.0, 25.0])
@pytest.mark.parametrize("width", [0, 2048], ids=["whole", "shared"])
def test_infinite_values_far_below_the_largest(width: int, gap: float, dtype: torch.dtype, device: torch.device) -> None:
    """An infinite value at exp(-gap) = 2^-36 of the largest probability is infinite in its channel and in no other."""
    for n, leader, inf in ((31, 30, 7), (900, 0, 7), (900, 7, 7)):
        out = _call(device, n, gap, leader, dtype, False, width, inf)[0]
        assert (out[0, :GROUP, 5] == float("inf")).all()
        rest = out.clone()
        rest[0, :GROUP, 5] = 0.0
        assert torch.isfinite(rest).all()


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [8.0, 22.0])
def test_host_route_and_the_bound(gap: float, dtype: torch.dtype, fp8: bool) -> None:
    """The host route keeps to the bound without the halves' share; a result off by 1% is outside it."""
    out, q, c, table = _call(torch.device("cpu"), 31, gap, 30, dtype, fp8, 0)
    _check(out, q, c, table, 31, fp8)
    with pytest.raises(AssertionError):
        _check(out.double() * 1.01, q, c, table, 31, fp8)
