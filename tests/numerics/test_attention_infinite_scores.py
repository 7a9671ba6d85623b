"""The paged attention where every token that takes part scores -infinity: 0 / 0, NaN, on the GPU as on the host; where no
token takes part, zeros; and where one token scores more, that token's value."""

from __future__ import annotations

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import kv_cases as kc

ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]
HEADS = 2


def _check(device: torch.device, dtype: torch.dtype, fp8: bool, page: int, width: int, d: int, group: int, window: int) -> None:
    # all of a head's scores -infinity in sequences 0, 2 and 4; 1 ordinary; of 3 no page is there, of 4 not all; 5 empty
    lens = [31, 90, 700, 40, 200, 0]
    table, pages = kc.tables(lens, page, width)
    c = kc.cache(pages, HEADS, page, d, dtype, fp8)
    for b in (0, 2, 4):
        for p in table[b, : -(-lens[b] // page)].tolist():
            if fp8:  # codes below zero times a scale without end
                c.k[p, 1] = torch.full((page, d), -1.0).to(kc.F8)
                c.ks[p, 1] = float("inf")
            else:
                c.k[p, 1, :, 0] = float("-inf")
    table[3] = -1
    table[4, 1] = -1
    q = torch.ones((6, HEADS * group, d), dtype=dtype)
    args = [t if t is None else t.to(device) for t in (q, *c.to("cpu"), table, torch.tensor(lens, dtype=torch.int32))]
    out = ops.paged_attention(*args, 0.01, window).cpu()
    for b in range(6):
        if b in (0, 2, 4):
            assert torch.isnan(out[b, group:]).all() and torch.isfinite(out[b, :group]).all() and out[b, :group].any()
        else:
            assert torch.isfinite(out[b]).all() and bool(out[b].any()) == (b == 1)
    # one token of each that scores more (within every window): its value alone
    for b in (0, 2, 4):
        i = lens[b] - 1
        at, off = int(table[b, i // page]), i % page
        if fp8:
            c.ks[at, 1, off] = 1e-3
        else:
            c.k[at, 1, off, 0] = 0.0
    cache = [t if t is None else t.to(device) for t in c.to("cpu")]
    out = ops.paged_attention(args[0], *cache, *args[5:], 0.01, window).cpu()
    for b in (0, 2, 4):
        i = lens[b] - 1
        at, off = int(table[b, i // page]), i % page
        want = c.v[at, 1, off].float() * (c.vs[at, 1, off] if fp8 else 1.0)
        # the probability is 1: two halves within 2^-16 of it, e4m3's scale in them, one rounding (fp16's subnormal step)
        assert ((out[b, group:].float() - want).abs() <= want.abs() * (2.0**-15 + kc.EPS[dtype]) + 2.0**-25).all()


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("window", [0, 25])
def test_host(window: int, dtype: torch.dtype, fp8: bool) -> None:
    _check(torch.device("cpu"), dtype, fp8, 16, 0, 64, 3, window)


@pytest.mark.gpu
@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("window", [0, 25])
@pytest.mark.parametrize(("d", "group"), [(64, 3), (80, 20), (128, 7), (256, 2)])
@pytest.mark.parametrize(("page", "width"), [(16, 0), (24, 0), (16, 2048), (24, 1400)])
def test_gpu(page: int, width: int, d: int, group: int, window: int, dtype: torch.dtype, fp8: bool,
             device: torch.device) -> None:
    _check(device, dtype, fp8, page, width, d, group, window)
