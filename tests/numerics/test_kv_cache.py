"""Writing and reading the paged cache on the GPU against the definitions, at the sizes, layouts, slots and values
where they can go wrong.

Bounds. The rotation is two products and a sum in fp32: within 3 * 2^-24 of |a| + |b| of a pair (|cos|, |sin| <= 1),
then half a step of the 16-bit value. Codes of unrotated rows equal the framework's quantizer on the host bit for bit;
a rotated row's scale is within that error of its largest value (and a rounding), and its codes within half a step of
the value over the scale that was returned, widened by the error.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.library import opcheck

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from oracle import fp8_block as oblk
from oracle import kv_cache as okv
from tests.numerics import kv_cases as kc
from tokenforge.kernels import host

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]


def _rows(t: int, heads: int, d: int, dtype: torch.dtype, seed: int) -> torch.Tensor:
    x = torch.randn((t, heads, d), generator=kc.gen("rows", t, heads, d, seed))
    x[..., :: max(1, d // 4)] *= 8.0
    return x.to(dtype)


def _slots(t: int, pages: int, page: int, seed: int = 0) -> torch.Tensor:
    return torch.randperm(pages * page, generator=kc.gen("slots", t, pages, page, seed))[:t]


def _table(rot: int, far: int) -> torch.Tensor:
    freq = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(far, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _bits(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous().cpu()
    return x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def _same(a, b) -> None:  # type: ignore[no-untyped-def]
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        assert x is None or torch.equal(_bits(x), _bits(y))


SIZES = [(1, 4, 128, 16), (1, 2, 64, 16), (7, 1, 256, 8), (33, 3, 80, 5), (5, 12, 72, 1), (130, 2, 8, 24), (4, 1, 248, 64),
         (3, 5, 136, 16), (2050, 4, 128, 16)]


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("tokens_first", [False, True])
@pytest.mark.parametrize(("t", "heads", "d", "page"), SIZES)
def test_write_and_read(t: int, heads: int, d: int, page: int, tokens_first: bool, dtype: torch.dtype, fp8: bool,
                        device: torch.device) -> None:
    """Every bit of the cache as the host's expression leaves it, what is not written untouched; and read back."""
    pages = t // page + 3
    c = kc.cache(pages, heads, page, d, dtype, fp8, tokens_first=tokens_first)
    k, v, slots = _rows(t, heads, d, dtype, 1), _rows(t, heads, d, dtype, 2), _slots(t, pages, page)
    if t > 3:
        slots[[0, 2, 3]] = torch.tensor([-1, pages * page, 2**62])  # padding and slots of no page
    dev = c.to(device)
    assert ops.kv_cache_write(k.to(device), v.to(device), *dev, slots.to(device)) is None
    host.kv_cache_write(k.float(), v.float(), c.k, c.v, c.ks, c.vs, slots)
    _same(dev, (c.k, c.v, c.ks, c.vs))
    for out in (torch.float16, torch.bfloat16) if fp8 else (dtype,):
        got = ops.kv_cache_read(*dev, slots.to(device), out)
        _same(got, host.kv_cache_read(c.k, c.v, c.ks, c.vs, slots, out))
        for x, cache, scale in zip(got, (c.k, c.v), (c.ks, c.vs)):
            for i in range(t)[:40]:
                s = int(slots[i])
                if not 0 <= s < pages * page:
                    assert not x[i].any()
                    continue
                want = kc.values(cache.float()[s // page, :, s % page])
                want = want if scale is None else want * kc.values(scale[s // page, :, s % page])[:, None]
                # a product in fp32, then half a step (of fp16's subnormals)
                bound = kc.EPS[out] * np.abs(want) * (1 + 2.0**-8) + 2.0**-25
                assert (np.abs(kc.values(x[i]) - want) <= bound).all()


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("t", "q_heads", "heads", "d", "rot"), [
    (1, 28, 4, 128, 128), (5, 14, 2, 64, 64), (3, 3, 3, 128, 64), (9, 8, 1, 256, 256), (4, 2, 2, 80, 80),
    (6, 4, 2, 80, 20), (2, 2, 1, 96, 2), (3, 1, 1, 8, 6), (33, 5, 5, 72, 24), (700, 6, 2, 192, 96)])
def test_rope_write(t: int, q_heads: int, heads: int, d: int, rot: int, interleaved: bool, dtype: torch.dtype,
                    fp8: bool, device: torch.device) -> None:
    page, far = 16, 5000
    pages = t // page + 2
    c = kc.cache(pages, heads, page, d, dtype, fp8)
    q, k, v = (_rows(t, h, d, dtype, i) for i, h in enumerate((q_heads, heads, heads)))
    slots = _slots(t, pages, page)
    positions = torch.randint(0, far, (t,), generator=kc.gen("pos", t))
    positions[0] = far - 1
    table = _table(rot, far)
    dev = c.to(device)
    got = ops.rope_kv_cache_write(q.to(device), k.to(device), v.to(device), table.to(device), positions.to(device),
                                  *dev, slots.to(device), interleaved)
    assert got.shape == q.shape and got.dtype == dtype

    def turned(x: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
        """The rotated values in 64 bits, and the error of fp32's: 3 roundings of |a| + |b| at most."""
        y = okv.rotate(kc.values(x), table.numpy(), positions.numpy(), interleaved)
        size = np.abs(kc.values(x))
        z = size[..., :rot]
        pairs = z.reshape(*z.shape[:-1], -1, 2).sum(-1) if interleaved else z[..., :rot // 2] + z[..., rot // 2:]
        err = np.zeros_like(y)
        err[..., :rot] = np.repeat(pairs, 2, -1) if interleaved else np.concatenate([pairs, pairs], -1)
        return y, err * 3 * kc.U32

    def check16(x: torch.Tensor, y: np.ndarray, err: np.ndarray) -> None:
        bound = err + kc.EPS[dtype] * (np.abs(y) + err) + (2.0**-25 if dtype == torch.float16 else 0.0)
        assert (np.abs(kc.values(x) - y) <= bound).all()
        assert torch.equal(x[..., rot:], (x.new_tensor(y).to(x.dtype))[..., rot:])

    check16(got.cpu(), *turned(q))
    at, off = slots // page, slots % page
    kd, vd, ksd, vsd = (None if x is None else x.cpu() for x in dev)
    y, err = turned(k)
    if fp8:
        s = kc.values(ksd[at, :, off])
        want = oblk.block_scales(y.reshape(-1, d), 0).reshape(t, heads)
        assert (np.abs(s - want) <= err.max(-1) / 448 + 2 * kc.U32 * want).all()
        code = kc.values(kd.view(torch.uint8)[at, :, off].view(kc.F8).float())
        ratio = y / s[..., None]
        assert (np.abs(code - ratio) <= oblk.half_step(ratio) * (1 + 2.0**-20) + err / s[..., None] + 2.0**-20).all()
    else:
        check16(kd[at, :, off], y, err)
    # values are not turned, and nothing else is written
    plain = kc.cache(pages, heads, page, d, dtype, fp8)
    host.kv_cache_write(k.float(), v.float(), plain.k, plain.v, plain.ks, plain.vs, slots)
    _same((vd, vsd), (plain.v, plain.vs))
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    before = c.k.transpose(1, 2).reshape(pages * page, heads, d).view(torch.uint8)
    assert torch.equal(kd.transpose(1, 2).reshape(pages * page, heads, d).view(torch.uint8)[rest], before[rest])


@pytest.mark.parametrize("fp8", [False, True])
def test_positions_outside_the_table_and_padding(fp8: bool, device: torch.device) -> None:
    dtype, page, d = torch.bfloat16, 16, 128
    c = kc.cache(3, 2, page, d, dtype, fp8)
    q, k, v = _rows(5, 4, d, dtype, 0), _rows(5, 2, d, dtype, 1), _rows(5, 2, d, dtype, 2)
    table = _table(64, 100)
    positions = torch.tensor([99, 100, -1, 2**62, 7])
    slots = torch.tensor([-1, -1, -5, 48, 40])
    for interleaved in (False, True):
        dev = c.to(device)
        got = ops.rope_kv_cache_write(q.to(device), k.to(device), v.to(device), table.to(device),
                                      positions.to(device), *dev, slots.to(device), interleaved).cpu()
        assert torch.isnan(got[1:4, :, :64]).all() and torch.equal(got[:, :, 64:], q[:, :, 64:])
        assert torch.isfinite(got[[0, 4]]).all()
        want = c.to("cpu")
        kf = host.rotate(k.float(), table, positions, interleaved)
        host.kv_cache_write(kf, v.float(), *want, slots)
        changed = [(_bits(a) != _bits(b)).flatten(3 if a.dim() == 4 else 2).nonzero()[:, [0, 2]] for a, b in
                   zip([x for x in dev if x is not None], [x for x in c.to("cpu") if x is not None])]
        for at in changed:
            assert at.numel() and (at == torch.tensor([2, 8])).all()
        _same((dev[1], dev[3]), (want[1], want[3]))
    # a key turned by a position that the table lacks is NaN where it is turned, and in 8 bits in its row
    dev = c.to(device)
    ops.rope_kv_cache_write(q.to(device), k.to(device), v.to(device), table.to(device), positions.to(device), *dev,
                            torch.arange(5, device=device), False)
    row = dev[0][0, :, 1].float().cpu()
    assert torch.isnan(row if fp8 else row[:, :64]).all()


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
def test_layouts(dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Joined projections, tokens and heads exchanged, rows off 16 bytes, one row for all; slots and tables strided;
    keys and values in one tensor: the results of contiguous copies."""
    t, heads, d, page, pages = 40, 2, 128, 16, 5
    c = kc.cache(pages, heads, page, d, dtype, fp8)
    q, k, v = (_rows(t, h, d, dtype, i).to(device) for i, h in enumerate((6, heads, heads)))
    slots, positions = _slots(t, pages, page).to(device), torch.arange(t, device=device) + 5
    table = _table(d, 64).to(device)
    want = c.to(device)
    turned = ops.rope_kv_cache_write(q, k, v, table, positions, *want, slots, False)

    def same(q, k, v, table, positions, dev, slots) -> None:  # type: ignore[no-untyped-def]
        got = ops.rope_kv_cache_write(q, k, v, table, positions, *dev, slots, False)
        _same([got], [turned])
        _same(dev, want)
        _same(ops.kv_cache_read(*dev, slots, dtype), ops.kv_cache_read(*want, slots.contiguous(), dtype))

    joined = torch.cat([q, k, v], 1).flatten(1)
    parts = [x.unflatten(1, (-1, d)) for x in joined.split((6 * d, heads * d, heads * d), 1)]
    same(*parts, table, positions, c.to(device), slots)
    same(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)), table, positions, c.to(device), slots)
    off = [torch.cat([x[..., :3], x], -1)[..., 3:] for x in (q, k, v)]
    same(*off, table, positions, c.to(device), slots)
    wide = torch.cat([table, table], 1)[:, :d]
    same(q, k, v, wide, positions.repeat_interleave(2)[::2], c.to(device), slots.repeat_interleave(2)[::2])
    k1, v1, ks, vs = c.to(device)
    both = torch.stack([k1.view(torch.uint8), v1.view(torch.uint8)], 3).view(k1.dtype)
    same(q, k, v, table, positions, (both[..., 0, :], both[..., 1, :], ks, vs), slots)
    c.tokens_first = True
    same(q, k, v, table, positions, c.to(device), slots)
    one = k[:1].expand(t, -1, -1)
    a, b = c.to(device), c.to(device)
    ops.kv_cache_write(one, one, *a, slots)
    ops.kv_cache_write(one.contiguous(), one.contiguous(), *b, slots)
    _same(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_zeros_extremes_and_nan(dtype: torch.dtype, device: torch.device) -> None:
    x = torch.zeros((5, 2, 128), dtype=dtype)
    x[1, 0], x[1, 1] = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x[2, 0, 5], x[2, 1, 6], x[3, 0, 7] = float("nan"), float("inf"), float("-inf")
    x[4] = -x[1]
    for fp8 in (True, False):
        c = kc.cache(1, 2, 16, 128, dtype, fp8)
        dev = c.to(device)
        slots = torch.arange(5) * 3
        ops.kv_cache_write(x.to(device), x.to(device), *dev, slots.to(device))
        host.kv_cache_write(x.float(), x.float(), c.k, c.v, c.ks, c.vs, slots)
        for a, b in zip(dev, (c.k, c.v, c.ks, c.vs)):
            if a is not None:
                assert torch.equal(torch.nan_to_num(a.float().cpu(), 999.0), torch.nan_to_num(b.float(), 999.0))
        if fp8:  # a row's NaN stays in it
            assert torch.isnan(dev[0][0, 0, 6].float()).any()
            assert torch.isfinite(dev[0][0, :, [0, 3, 12]].float()).all()
        _, v = ops.kv_cache_read(*dev, slots.to(device), dtype)
        _, vh = host.kv_cache_read(c.k, c.v, c.ks, c.vs, slots, dtype)
        assert torch.equal(torch.nan_to_num(v.cpu(), 9.0), torch.nan_to_num(vh, 9.0))


def test_every_code_is_read_exactly(device: torch.device) -> None:
    codes = torch.arange(256, dtype=torch.uint8).reshape(1, 2, 1, 128)
    k = codes.view(kc.F8).to(device)
    for s in (1.0, 3.1e-3, 2.0**-18, 1e4):
        scale = torch.full((1, 2, 1), s, device=device)
        for out in (torch.float16, torch.bfloat16):
            got = ops.kv_cache_read(k, k, scale, scale, torch.zeros(1, dtype=torch.int64, device=device), out)[0].cpu()
            want = (codes.view(kc.F8).float() * torch.tensor(s)).to(out).reshape(1, 2, 128)
            assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0))


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_past_32_bits(fp8: bool, device: torch.device) -> None:
    dtype, page, d, heads = torch.float16, 16, 128, 2
    c = kc.cache(2, heads, page, d, dtype, fp8)
    far = (1 << 32) // (heads * page * d) + 3
    big = [None if t is None else torch.empty((far + 2, *t.shape[1:]), dtype=t.dtype, device=device)
           for t in (c.k, c.v, c.ks, c.vs)]
    k, v = _rows(20, heads, d, dtype, 1), _rows(20, heads, d, dtype, 2)
    slots = torch.arange(20) + 5
    for x, t in zip(big, (c.k, c.v, c.ks, c.vs)):
        if x is not None:
            x[far:] = t.to(device)
    ops.kv_cache_write(k.to(device), v.to(device), *big, (slots + far * page).to(device))
    host.kv_cache_write(k.float(), v.float(), c.k, c.v, c.ks, c.vs, slots)
    _same([None if x is None else x[far:] for x in big], (c.k, c.v, c.ks, c.vs))
    _same(ops.kv_cache_read(*big, (slots + far * page).to(device), dtype),
          host.kv_cache_read(c.k, c.v, c.ks, c.vs, slots, dtype))


@pytest.mark.parametrize("page", [32, 24])
def test_slots_past_31_bits(page: int, device: torch.device) -> None:
    """Slot numbers up to 2^33 (a page repeated 2^28 times)."""
    one = torch.randn((1, 2, page, 64), generator=kc.gen("repeated")).half()
    pages = 1 << 28
    cache = one.to(device).expand(pages, -1, -1, -1)
    slots = torch.tensor([0, 2**31 - 1, 2**31, 2**31 + 7, 2**32 + 5, pages * page - 1, pages * page, 2**31 - page, 5 * page])
    k, v = ops.kv_cache_read(cache, cache, None, None, slots.to(device), torch.float16)
    want = one[0, :, slots % page].transpose(0, 1).clone()
    want[6] = 0
    assert torch.equal(k.cpu(), want) and torch.equal(v, k)


def test_many_tokens(device: torch.device) -> None:
    """Tens of thousands of tokens; and more rows than a launch takes (2^26), written, rotated and read in parts."""
    t, heads, d, page = 20000, 12, 64, 128
    pages = t // page + 1
    k = torch.randn((1, heads, d), device=device).half().expand(t, heads, d)
    v = k + torch.arange(t, device=device).half()[:, None, None] / 64
    dev = kc.cache(pages, heads, page, d, torch.float16, True).to(device)
    slots = torch.arange(t, device=device)
    ops.kv_cache_write(k, v, *dev, slots)
    for x, got in zip((k, v), ops.kv_cache_read(*dev, slots, torch.float16)):
        top = x.float().abs().amax(-1, keepdim=True)
        assert ((got.float() - x.float()).abs() <= top * (2.0**-4 + 2.0**-8)).all()
    del dev
    t, heads, d, page = 2500, 16384, 8, 50  # 2048 tokens a launch; with as many queries 1365
    x = torch.randn((t, 1, d), device=device).bfloat16()
    k, slots = x.expand(t, heads, d), torch.arange(t, device=device).flip(0)
    cache = [torch.zeros((t // page, heads, page, d), dtype=torch.bfloat16, device=device) for _ in "kv"]
    ops.kv_cache_write(k, -k, *cache, None, None, slots)
    got = ops.kv_cache_read(*cache, None, None, slots, torch.bfloat16)
    assert torch.equal(got[0], k) and torch.equal(got[1], -k)
    quarter = torch.tensor([[0.0] * 4 + [1.0] * 4], device=device)  # a quarter turn: (a, b) -> (-b, a)
    q = ops.rope_kv_cache_write(-k, k, k, quarter, torch.zeros_like(slots), *cache, None, None, slots)
    turned = torch.cat([-x[..., 4:], x[..., :4]], -1).expand(t, heads, d)
    assert torch.equal(q, -turned)
    del q, got
    got = ops.kv_cache_read(*cache, None, None, slots, torch.bfloat16)
    assert torch.equal(got[0], turned) and torch.equal(got[1], k)


def test_graphs_streams_and_opcheck(device: torch.device) -> None:
    t, heads, d, page, dtype = 6, 2, 64, 16, torch.bfloat16
    c = kc.cache(4, heads, page, d, dtype, True)
    q, k, v = (_rows(t, h, d, dtype, i).to(device) for i, h in enumerate((4, heads, heads)))
    table, positions = _table(d, 100).to(device), torch.arange(t, device=device)
    slots = torch.arange(t, device=device) * 2
    dev, eager = c.to(device), c.to(device)
    graph = torch.cuda.CUDAGraph()
    ops.rope_kv_cache_write(q, k, v, table, positions, *dev, slots, False)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.rope_kv_cache_write(q, k, v, table, positions, *dev, slots, False)
        back = ops.kv_cache_read(*dev, slots, dtype)
    ops.rope_kv_cache_write(q, k, v, table, positions, *eager, slots, False)
    for step in range(4):
        slots += 1
        positions.copy_((positions * 3 + step) % 100)
        graph.replay()
        want = ops.rope_kv_cache_write(q, k, v, table, positions, *eager, slots, False)
        torch.cuda.synchronize()
        _same([out, *dev], [want, *eager])
        _same(back, ops.kv_cache_read(*eager, slots, dtype))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.kv_cache_write(k, v, *dev, slots)
    stream.synchronize()
    ops.kv_cache_write(k, v, *eager, slots)
    _same(dev, eager)
    for fp8 in (False, True):
        # test_schema multiplies its inputs, which e4m3 lacks
        only = {"test_utils": "test_faketensor"} if fp8 else {}
        x = kc.cache(4, heads, page, d, dtype, fp8)
        opcheck(ops.kv_cache_write, (k, v, *x.to(device), slots), **only)
        opcheck(ops.rope_kv_cache_write, (q, k, v, table, positions, *x.to(device), slots, True), **only)
        opcheck(ops.kv_cache_read, (*x.to(device), slots, dtype), **only)

    def step_fn(k, v, a, b, x, y, s):  # type: ignore[no-untyped-def]
        ops.kv_cache_write(k, v, a, b, x, y, s)
        return ops.kv_cache_read(a, b, x, y, s, torch.bfloat16)[0] * 2

    mine = c.to(device)
    got = torch.compile(step_fn, fullgraph=True, backend="aot_eager")(k, v, *mine, slots)
    other = c.to(device)
    assert torch.equal(got, step_fn(k, v, *other, slots))
    _same(mine, other)
