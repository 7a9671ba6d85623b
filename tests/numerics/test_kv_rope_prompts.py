"""The rotation and write of prompts long enough (16384 rows) that a lane group takes two rows with one load of their angles:
keys and values in one group (an odd number of heads), a last row alone (an odd number of rows), rotations by halves,
in pairs and an element at a time, of the whole head and of its part. Bounds: ``test_kv_cache.test_rope_write``."""

from __future__ import annotations

import pytest
import torch

from tests.numerics import test_kv_cache as short

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize(("dtype", "fp8"), short.TYPES, ids=short.IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("t", "q_heads", "heads", "d", "rot"), [
    (500, 28, 4, 128, 128), (1500, 7, 2, 64, 64), (1300, 7, 3, 128, 128), (1700, 6, 2, 192, 96), (1500, 5, 3, 256, 256),
    (2100, 4, 2, 80, 20), (1500, 5, 3, 56, 16), (1500, 9, 1, 72, 24), (5500, 1, 1, 40, 32)])
def test_rope_write_of_long_prompts(t: int, q_heads: int, heads: int, d: int, rot: int, interleaved: bool, dtype: torch.dtype,
                                    fp8: bool, device: torch.device) -> None:
    assert t * (q_heads + 2 * heads) >= 16384
    short.test_rope_write(t, q_heads, heads, d, rot, interleaved, dtype, fp8, device)
