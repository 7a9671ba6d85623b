"""The cache's writes advance the version counters of what they write, as torch's own do: a gradient that saved a cache
which was written since is refused."""

from __future__ import annotations

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import kv_cases as kc

ops = torch.ops.tokenforge
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device: str, fp8: bool, cache, even: bool):  # type: ignore[no-untyped-def]
    rows = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=device)
    slots = torch.arange(3, device=device)
    if not even:  # a form that the GPU's short path leaves to the Python body
        slots = slots.repeat_interleave(2)[::2]
    cos_sin = torch.ones((4, 64), device=device)
    yield lambda: ops.kv_cache_write(rows, rows, *cache, slots)
    yield lambda: ops.rope_kv_cache_write(rows, rows, rows, cos_sin, slots, *cache, slots)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("even", [False, True])
def test_written_tensors_count(even: bool, fp8: bool, device: str) -> None:
    cache = kc.cache(2, 2, 16, 64, torch.bfloat16, fp8).to(device)
    held = [t for t in cache if t is not None]
    slots = torch.arange(3, device=device)
    for call in _calls(device, fp8, cache, even):
        before = [t._version for t in held]
        call()
        assert all(t._version > n for t, n in zip(held, before))
    before = [t._version for t in held]
    ops.kv_cache_read(*cache, slots, torch.bfloat16)
    q = torch.ones((1, 2, 64), dtype=torch.bfloat16, device=device)
    ops.paged_attention(q, *cache, torch.zeros((1, 1), dtype=torch.int32, device=device),
                        torch.ones(1, dtype=torch.int32, device=device), 1.0)
    assert before == [t._version for t in held]


@pytest.mark.parametrize("device", DEVICES)
def test_a_saved_cache_that_was_written_is_refused(device: str) -> None:
    cache = kc.cache(2, 2, 16, 64, torch.bfloat16, False).to(device)
    weight = torch.ones(64, dtype=torch.bfloat16, device=device, requires_grad=True)
    for call in _calls(device, False, cache, True):
        y = (cache[0] * weight).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("even", [False, True])
def test_inference_tensors_are_written(even: bool) -> None:
    """A cache made under inference mode is written inside and outside of it, as before; one made outside counts in both."""
    with torch.inference_mode():
        cache = kc.cache(2, 2, 16, 64, torch.bfloat16, True).to("cuda")
        for call in _calls("cuda", True, cache, even):
            call()
    for call in _calls("cuda", True, cache, even):
        call()
    assert cache[0].view(torch.uint8).any() and cache[0].is_inference()
    cache = kc.cache(2, 2, 16, 64, torch.bfloat16, True).to("cuda")
    with torch.inference_mode():
        before = [t._version for t in cache]
        for call in _calls("cuda", True, cache, even):
            call()
    assert all(t._version > n for t, n in zip(cache, before))
