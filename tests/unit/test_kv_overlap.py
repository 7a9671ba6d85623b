"""A written cache's keys, values and scales lie apart: what overlaps is refused by the operators and by the C entries, what
is only interleaved is not."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import kv_cases as kc
from tokenforge.kernels import _lib
from tokenforge.kernels.hip import kv_cache as kv

ops = torch.ops.tokenforge
PAGES, HEADS, PAGE, D = 3, 2, 16, 64


def _write(k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor | None = None, vs: torch.Tensor | None = None) -> None:
    dev = k.device
    dtype = torch.float16 if ks is not None else k.dtype
    rows = torch.ones((2, k.shape[1], k.shape[3]), dtype=dtype, device=dev)
    slots = torch.arange(2, device=dev)
    ops.kv_cache_write(rows, rows, k, v, ks, vs, slots)
    cos_sin = torch.ones((4, k.shape[3]), device=dev)
    ops.rope_kv_cache_write(rows, rows, rows, cos_sin, slots, k, v, ks, vs, slots)


def _overlapping(device: torch.device | str) -> list[tuple]:  # type: ignore[type-arg]
    flat = torch.zeros(4 * PAGES * HEADS * PAGE * D, dtype=torch.float16, device=device)
    size, strides = PAGES * HEADS * PAGE * D, (HEADS * PAGE * D, PAGE * D, D, 1)
    shape = (PAGES, HEADS, PAGE, D)

    def at(offset: int, st: tuple[int, ...] = strides) -> torch.Tensor:
        return flat.as_strided(shape, st, offset)

    f8 = torch.zeros(4 * size, dtype=torch.uint8, device=device)
    scales = torch.ones(4 * PAGES * HEADS * PAGE, device=device)

    def codes(offset: int) -> torch.Tensor:
        return f8.as_strided(shape, strides, offset).view(kc.F8)

    def scale(offset: int) -> torch.Tensor:
        return scales.as_strided(shape[:3], (HEADS * PAGE, PAGE, 1), offset)

    inside = f8.view(torch.float32).as_strided(shape[:3], (HEADS * PAGE, PAGE, 1), 16)
    wide = (2 * HEADS * PAGE * D, PAGE * D, D, 1)
    return [
        (at(0), at(D)),  # a row further
        (at(0), at(size - D)),  # the last row and the first
        (at(size - 8), at(0)),
        (at(0, wide), at(HEADS * PAGE * D - 8, wide)),  # pages side by side, by a piece too near
        (at(0), at(PAGE * D, (PAGE * HEADS * D, D, HEADS * D, 1))),  # by head and then token, by token and then head
        (codes(0), codes(8), scale(0), scale(PAGES * HEADS * PAGE)),
        (codes(0), codes(size), scale(0), scale(1)),
        (codes(0), codes(size), inside, scale(0)),  # keys' scales among the keys' codes
        (codes(size), codes(0), scale(0), inside),
    ]


def _apart(device: torch.device | str) -> list[tuple]:  # type: ignore[type-arg]
    both = torch.zeros((PAGES, HEADS, PAGE, 2, D), dtype=torch.float16, device=device)
    pages = torch.zeros((PAGES, 2, HEADS, PAGE, D), dtype=torch.float16, device=device)
    first = torch.zeros((2, PAGES, HEADS, PAGE, D), dtype=torch.float16, device=device)
    mixed = torch.zeros((PAGES, 2, HEADS * PAGE * D), dtype=torch.float16, device=device)
    heads = torch.zeros((PAGES, PAGE, 2 * HEADS, D), dtype=torch.float16, device=device)
    # a row of codes, its scale and four bytes of nothing, keys and values in turn
    rows = torch.zeros((PAGES, PAGE, HEADS, 2, D + 8), dtype=torch.uint8, device=device).permute(0, 2, 1, 3, 4)
    c = [rows[..., i, :D].view(kc.F8) for i in range(2)]
    s = [rows[..., i, D:D + 4].view(torch.float32)[..., 0] for i in range(2)]
    pair = torch.ones((PAGES, HEADS, PAGE, 2), device=device)
    lone = torch.zeros((2, 1, 1, 1, D), dtype=torch.float16, device=device)
    return [
        (both[..., 0, :], both[..., 1, :]), (both[..., 1, :], both[..., 0, :]),
        (pages[:, 0], pages[:, 1]), (first[0], first[1]),
        (mixed[:, 0].unflatten(1, (HEADS, PAGE, D)), mixed[:, 1].unflatten(1, (PAGE, HEADS, D)).transpose(1, 2)),
        (heads[:, :, :HEADS].transpose(1, 2), heads[:, :, HEADS:].transpose(1, 2)),
        (*c, *s), (c[1], c[0], s[0], s[1]), (*c, pair[..., 0], pair[..., 1]),
        (lone[0], lone[1]),
    ]


@pytest.mark.parametrize("device_name", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_what_overlaps_is_refused_and_what_is_interleaved_is_not(device_name: str) -> None:
    for case in _overlapping(device_name):
        before = [t.clone() for t in case]
        with pytest.raises(ValueError, match="overlap"):
            _write(*case)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(case, before) if a.element_size() == 1)
        assert not case[0].view(torch.uint8).any()  # nothing was written
    for case in _apart(device_name):
        _write(*case)
        assert case[0].view(torch.uint8)[0, :, :2].any() and case[1].view(torch.uint8)[0, :, :2].any()


def _c_refuses(k: int, v: int, ks: int, vs: int, shape: tuple[int, ...], strides: list[tuple[int, ...]]) -> bool:
    """Whether the C entry refuses to write into such a cache of e4m3 codes (a call of no tokens: nothing is launched)."""
    three = ctypes.c_int64 * 3
    c = _lib.TfKvCache(k, v, ks, vs, *shape, _lib.DTYPE_E4M3, *(three(*s) for s in strides))
    h = _lib.lib()
    rc = h.tf_kv_cache_write(ctypes.byref(c), 1 << 40, 0, 0, 1 << 41, 0, 0, 0, 1 << 42, 0, None)
    if rc != _lib.TF_OK:
        assert rc == _lib.TF_EINVAL and (b"overlap" in h.tf_last_error() or b"one place" in h.tf_last_error())
    return rc != _lib.TF_OK


def _bytes(at: int, strides: tuple[int, ...], shape: tuple[int, ...], run: int) -> set[int]:
    out = {at}
    for st, n in zip(strides, shape):
        out = {a + st * i for a in out for i in range(n)}
    return {a + i for a in out for i in range(run)}


def _nested(rng: random.Random, shape: tuple[int, ...], run: int, step: int) -> tuple[int, ...]:
    """Byte strides that keep rows of ``run`` bytes apart, multiples of ``step``, the dimensions in any order."""
    order, out, extent = rng.sample(range(3), 3), [0, 0, 0], run
    for i in order:
        out[i] = -(-(extent + rng.choice((0, 0, step, 2 * step))) // step) * step
        extent += out[i] * (shape[i] - 1)
    return tuple(out)


@pytest.mark.parametrize("seed", range(40))
def test_against_every_byte(seed: int) -> None:
    """Drawn layouts: what shares a byte is always refused, by Python and C alike; what does not is taken where the strides
    are the same or the ranges apart."""
    rng = random.Random(seed)
    pool = torch.zeros(1 << 16, dtype=torch.uint8)
    base = pool.data_ptr()
    for _ in range(40):
        shape, d = tuple(rng.randint(1, 3) for _ in range(3)), 8 * rng.randint(1, 2)
        k_st = _nested(rng, shape, d, 8)
        same = rng.random() < 0.6
        v_st = k_st if same else _nested(rng, shape, d, 8)
        v_at = 8 * rng.randint(0, 40)
        k_at = 8 * rng.randint(0, 40)
        kb, vb = _bytes(k_at, k_st, shape, d), _bytes(v_at, v_st, shape, d)
        far = 1 << 15
        s_st = _nested(rng, shape, 4, 4)
        scale_at = (far, far + 8192)
        k, v = (pool.as_strided((*shape, d), (*st, 1), at).view(kc.F8) for st, at in ((k_st, k_at), (v_st, v_at)))
        ks, vs = (pool.view(torch.float32).as_strided(shape, tuple(x // 4 for x in s_st), at // 4) for at in scale_at)
        refused = []
        try:
            kv.check_cache(k, v, ks, vs, written=True)
            refused.append(False)
        except ValueError as e:
            assert "overlap" in str(e) or "one tensor" in str(e)
            refused.append(True)
        refused.append(_c_refuses(base + k_at, base + v_at, base + scale_at[0], base + scale_at[1], (*shape, d),
                                  [k_st, v_st, tuple(x // 4 for x in s_st), tuple(x // 4 for x in s_st)]))
        assert refused[0] == refused[1]
        if kb & vb:
            assert refused[0]
        elif same or max(kb) < min(vb) or max(vb) < min(kb):
            assert not refused[0]
        # scales among codes of one buffer
        inside = 4 * rng.randint(0, 80)
        sb = _bytes(inside, s_st, shape, 4)
        got = _c_refuses(base + k_at, base + (1 << 14), base + inside, base + far, (*shape, d),
                         [k_st, k_st, tuple(x // 4 for x in s_st), tuple(x // 4 for x in s_st)])
        s_in = pool.view(torch.float32).as_strided(shape, tuple(x // 4 for x in s_st), inside // 4)
        v_far = pool.as_strided((*shape, d), (*k_st, 1), 1 << 14).view(kc.F8)
        try:
            kv.check_cache(k, v_far, s_in, ks, written=True)
            mine = False
        except ValueError:
            mine = True
        assert mine == got and (got or not kb & sb)
        if not got:
            continue
        assert not (max(kb) < min(sb) or max(sb) < min(kb))
