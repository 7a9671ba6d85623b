"""Which sizes the attention takes: the operators' check and the C entry agree, at and around every limit."""

from __future__ import annotations

import ctypes

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tokenforge.kernels import _lib
from tokenforge.kernels.hip import kv_cache as kv


def _takes(m: int, heads: int, group: int, page: int, width: int, d: int) -> bool:
    one = torch.zeros(1, dtype=torch.float16)
    k, v = (one.expand(d).contiguous().as_strided((1, heads, page, d), (0, 0, 0, 1)) for _ in "kv")
    q = one.expand(d).contiguous().as_strided((m, heads * group, d), (0, 0, 1))
    table = torch.zeros(1, dtype=torch.int32)
    try:
        kv.check_attention(q, (k, v, None, None), table.expand(m, width), table.expand(m), 0)
    except ValueError as e:
        assert "too large" in str(e)
        return False
    return True


def _c_takes(m: int, heads: int, group: int, page: int, width: int, d: int) -> bool:
    c = _lib.TfKvCache(1 << 20, 1 << 21, None, None, 1, heads, page, d, 0)
    return _lib.lib().tf_paged_attention_workspace_bytes(ctypes.byref(c), m, heads * group, width, 0) >= 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 16, 17, 32, 33, 300])
@pytest.mark.parametrize("heads", [1, 3])
@pytest.mark.parametrize("page", [16, 24, 1 << 20])
def test_the_check_and_the_c_entry_agree(page: int, heads: int, group: int, d: int) -> None:
    most = 0x7FFFFF00 // page
    for m in (1, 2, 5, 64):
        rows = m * heads * -(-group // (32 if group > 16 and d <= 128 else 16))
        edge = (0x7FFFFFFF // rows) * 16 // page  # tokens of a row that reach the limit on steps of 16
        for width in {0, 1, most, most + 1, edge - 1, edge, edge + 1, edge // 2, min(2 * edge, most)}:
            if width >= 0:
                assert _takes(m, heads, group, page, width, d) == _c_takes(m, heads, group, page, width, d), (m, width)


def test_many_query_heads_over_a_long_table() -> None:
    """Heads past 16 share their loads by 32, so such a table holds twice as many of them."""
    page, d, group = 1 << 20, 8, 300
    k, v = (torch.randn((1, 1, page, d), generator=torch.Generator().manual_seed(i)).half() for i in range(2))
    q = torch.ones((1, group, d), dtype=torch.float16)
    table = torch.zeros((1, 2046), dtype=torch.int32)
    out = torch.ops.tokenforge.paged_attention(q, k, v, None, None, table, torch.tensor([2], dtype=torch.int32), 0.1)
    p = torch.softmax(k[0, 0, :2].double().sum(1) * 0.1, 0)
    want = p @ v[0, 0, :2].double()
    # two tokens' sums in fp32, one rounding (2^-11) of a value of at most the values' magnitudes
    assert ((out.double() - want).abs() <= v[0, 0, :2].double().abs().amax(0) * 2.0**-10).all()
