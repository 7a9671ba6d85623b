"""The paged cache and its attention, the parts that need no GPU: the host route against the definitions in 64 bits,
refusals of the operators and of the C entry points, fakes, and the page division."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.library import opcheck

import tokenforge.kernels.ops  # noqa: F401
from oracle import kv_cache as okv
from tests.numerics import kv_cases as kc
from tokenforge.kernels import _lib
from tokenforge.kernels.hip import kv_cache as kv

ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]


def _rows(t: int, heads: int, d: int, dtype: torch.dtype, seed: int) -> torch.Tensor:
    return torch.randn((t, heads, d), generator=kc.gen("rows", t, heads, d, seed)).to(dtype)


# ----------------------------------------------------------------------------- host route


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize(("page", "window", "d"), [(16, 0, 64), (5, 0, 24), (16, 20, 128), (1, 7, 8)])
def test_host_attention(page: int, window: int, d: int, dtype: torch.dtype, fp8: bool) -> None:
    lens = [40, 0, 1, 33, 90]
    table, pages = kc.tables(lens, page)
    if window == 0:
        table[4, 2] = pages + 3  # a page that is not there
    c = kc.cache(pages, 2, page, d, dtype, fp8)
    q = _rows(5, 6, d, dtype, 0)
    out = ops.paged_attention(q, *c.to("cpu"), table, torch.tensor(lens, dtype=torch.int32), d**-0.5, window)
    assert out.dtype == dtype
    kc.check_attention(out, q, c, table, lens, d**-0.5, window)
    over = torch.tensor([2**31 - 1, -3, 1, 33, 90], dtype=torch.int32)
    out = ops.paged_attention(q, *c.to("cpu"), table, over, d**-0.5, window)
    kc.check_attention(out, q, c, table, [table.shape[1] * page, 0, 1, 33, 90], d**-0.5, window)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_host_write_and_read(interleaved: bool, dtype: torch.dtype, fp8: bool) -> None:
    t, heads, d, page, rot = 9, 2, 40, 4, 24
    c = kc.cache(5, heads, page, d, dtype, fp8)
    q, k, v = (_rows(t, h, d, dtype, i) for i, h in enumerate((6, heads, heads)))
    angle = torch.arange(50, dtype=torch.float64)[:, None] * 0.3 ** torch.arange(rot // 2)
    table = torch.cat([angle.cos(), angle.sin()], 1).float()
    positions = torch.arange(t) * 5
    slots = torch.randperm(20, generator=kc.gen("slots"))[:t]
    slots[2], slots[5] = -1, 20
    dev = c.to("cpu")
    got = ops.rope_kv_cache_write(q, k, v, table, positions, *dev, slots, interleaved)
    for x, have in ((q, got), (k, None)):
        want = okv.rotate(kc.values(x), table.numpy(), positions.numpy(), interleaved)
        if have is None:
            kept = (slots >= 0) & (slots < 20)
            have = ops.kv_cache_read(*dev, slots, dtype)[0]
            assert not have[~kept].any()
            have, want = have[kept], want[kept.numpy()]
        # the pair's sum of magnitudes is at most sqrt(2) of a rotated pair's largest: three roundings of it, half a
        # step in 16 bits, and half an e4m3 step (2^-4 of a value, 2^-10 of the largest's 448th part)
        top = np.abs(want).max(-1, keepdims=True)
        bound = 8 * kc.U32 * top + 2 * kc.EPS[dtype] * np.abs(want) + (2.0**-4 * np.abs(want) + 2.0**-17 * top) * fp8
        assert (np.abs(kc.values(have) - want) <= bound).all()
    plain = c.to("cpu")
    ops.kv_cache_write(k, v, *plain, slots)
    assert torch.equal(plain[1].view(torch.uint8), dev[1].view(torch.uint8))
    if not fp8:
        at = slots[(slots >= 0) & (slots < 20)]
        assert torch.equal(plain[1][at // page, :, at % page], v[(slots >= 0) & (slots < 20)])
    far = torch.tensor([0, 50, -1, 2**60, 1, 2, 3, 4, 5])
    got = ops.rope_kv_cache_write(q, k, v, table, far, *dev, torch.full((t,), -1), interleaved)
    assert torch.isnan(got[1:4, :, :rot]).all() and torch.isfinite(got[4:]).all()
    assert torch.equal(got[:, :, rot:], q[:, :, rot:])


def test_empty_calls() -> None:
    c = kc.cache(2, 2, 16, 64, torch.float16, True).to("cpu")
    x, s = torch.zeros((0, 2, 64), dtype=torch.float16), torch.zeros(0, dtype=torch.int64)
    assert ops.kv_cache_write(x, x, *c, s) is None
    assert ops.rope_kv_cache_write(x, x, x, torch.zeros((4, 64)), s, *c, s).shape == (0, 2, 64)
    assert ops.kv_cache_read(*c, s, torch.bfloat16)[1].shape == (0, 2, 64)
    none = torch.zeros((0, 3), dtype=torch.int32)
    assert ops.paged_attention(x, *c, none, none[:, 0], 1.0).shape == (0, 2, 64)
    q = torch.ones((2, 2, 64), dtype=torch.float16)
    assert not ops.paged_attention(q, *c, torch.zeros((2, 0), dtype=torch.int32), torch.ones(2, dtype=torch.int32),
                                   1.0).any()


def test_fakes_and_opcheck() -> None:
    with FakeTensorMode():
        c = [torch.empty((3, 2, 16, 64), dtype=kc.F8) for _ in "kv"] + [torch.empty((3, 2, 16)) for _ in "kv"]
        q, k = torch.empty((5, 4, 64), dtype=torch.bfloat16), torch.empty((5, 2, 64), dtype=torch.bfloat16)
        i = torch.empty(5, dtype=torch.int64)
        out = ops.rope_kv_cache_write(q, k, k, torch.empty((9, 32)), i, *c, i, True)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert [t.shape for t in ops.kv_cache_read(*c, i, torch.float16)] == [(5, 2, 64)] * 2
        assert ops.paged_attention(q, *c, torch.empty((5, 2), dtype=torch.int32), i.int(), 1.0).dtype == q.dtype
    c = kc.cache(3, 2, 16, 64, torch.float16, False).to("cpu")
    q, k, i = _rows(5, 4, 64, torch.float16, 0), _rows(5, 2, 64, torch.float16, 1), torch.arange(5)
    opcheck(ops.kv_cache_write, (k, k, *c, i))
    opcheck(ops.rope_kv_cache_write, (q, k, k, torch.ones((9, 32)), i, *c, i, False))
    opcheck(ops.kv_cache_read, (*c, i, torch.float16))
    opcheck(ops.paged_attention, (q, *c, torch.zeros((5, 2), dtype=torch.int32), i.int(), 1.0, 3))

    def step(q, k, v, cos_sin, pos, a, b, slots):  # type: ignore[no-untyped-def]
        q = ops.rope_kv_cache_write(q, k, v, cos_sin, pos, a, b, None, None, slots)
        return ops.paged_attention(q, a, b, None, None, slots[:, None].int() // 16, (slots % 16 + 1).int(), 0.1)

    args = (q, k, k, torch.ones((9, 32)), i)
    a, b = c[0].clone(), c[1].clone()
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(*args, c[0], c[1], i)
    assert torch.equal(got, step(*args, a, b, i)) and torch.equal(a, c[0]) and torch.equal(b, c[1])


# ----------------------------------------------------------------------------- refusals


def test_caches_are_refused() -> None:
    f16 = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    f8, s = torch.zeros((2, 2, 16, 64), dtype=kc.F8), torch.ones((2, 2, 16))
    slots = torch.arange(3)
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    long, far = torch.zeros((2, 2, 16, 264), dtype=torch.float16), torch.zeros((1 << 24) + 8)
    for error, match, cache in [
        (ValueError, "must be \\[pages", (f16[0], f16[0], None, None)),
        (ValueError, "v_cache shape", (f16, f16[:1], None, None)),
        (TypeError, "fp16, bf16 or float8", (f16.float(), f16.float(), None, None)),
        (TypeError, "v_cache must be", (f16, f16.bfloat16(), None, None)),
        (ValueError, "no slots", (f16[:0], f16[:0], None, None)),
        (ValueError, "head_dim", (f16[..., :12], f16[..., :12], None, None)),
        (ValueError, "head_dim", (long, long, None, None)),
        (ValueError, "head_dim", (f16[..., :0], f16[..., :0], None, None)),
        (ValueError, "go with", (f16, f16, s, s)),
        (ValueError, "go with", (f8, f8, s, None)),
        (ValueError, "k_scale shape", (f8, f8, s[:1], s)),
        (TypeError, "v_scale must be fp32", (f8, f8, s, s.half())),
        (ValueError, "contiguous in its last", (f16.transpose(2, 3)[..., :16], f16.transpose(2, 3)[..., :16], None, None)),
        (ValueError, "start on 16 bytes", (f16[..., 4:60], f16[..., 4:60], None, None)),
        (ValueError, "start on 16 bytes", (torch.zeros((2, 2, 16, 65), dtype=torch.float16)[..., :64], f16, None, None)),
        (ValueError, "elements apart", (far.half().as_strided((1, 1, 2, 8), (1 << 25, 1 << 25, 1 << 24, 1)),
                                        torch.zeros((1, 1, 2, 8), dtype=torch.float16), None, None)),
        (ValueError, "elements apart", (torch.zeros((1, 1, 2, 8), dtype=kc.F8), torch.zeros((1, 1, 2, 8), dtype=kc.F8),
                                        torch.ones((1, 1, 2)), far.as_strided((1, 1, 2), (1 << 25, 1 << 25, 1 << 24)))),
    ]:
        with pytest.raises(error, match=match):
            ops.kv_cache_read(*cache, slots, torch.float16)
        with pytest.raises(error, match=match):
            ops.kv_cache_write(x, x, *cache, slots)
        with pytest.raises(error, match=match):
            ops.paged_attention(x, *cache, torch.zeros((3, 1), dtype=torch.int32), slots.int(), 1.0)
    # a cache that is written holds each element once; one that is read may repeat
    twice, one = f16[:1].expand(2, -1, -1, -1), f16
    with pytest.raises(ValueError, match="twice"):
        ops.kv_cache_write(x, x, twice, one, None, None, slots)
    with pytest.raises(ValueError, match="twice"):
        ops.kv_cache_write(x, x, one, f16.as_strided((2, 2, 16, 64), (2048, 1024, 56, 1)), None, None, slots)
    with pytest.raises(ValueError, match="v_scale is written"):
        ops.kv_cache_write(x, x, f8, f8.clone(), s, s[..., :1].expand(2, 2, 16), slots)
    with pytest.raises(ValueError, match="one tensor"):
        ops.kv_cache_write(x, x, one, one, None, None, slots)
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        ops.kv_cache_write(x, x, f8, f8.clone(), s, s, slots)
    assert ops.kv_cache_read(one, one, None, None, slots, torch.float16)[0].shape == (3, 2, 64)
    assert ops.kv_cache_read(twice, one, None, None, slots, torch.float16)[0].shape == (3, 2, 64)


def test_writes_are_refused() -> None:
    c = (torch.zeros((2, 2, 16, 64), dtype=torch.float16), torch.zeros((2, 2, 16, 64), dtype=torch.float16), None, None)
    f8 = (c[0].to(kc.F8), c[1].to(kc.F8), torch.ones((2, 2, 16)), torch.ones((2, 2, 16)))
    x, q, slots = torch.zeros((3, 2, 64), dtype=torch.float16), torch.zeros((3, 4, 64), dtype=torch.float16), torch.arange(3)
    table = torch.zeros((9, 32))
    for error, match, k, v, cache, s in [
        (ValueError, "k must be", x[0], x, c, slots),
        (ValueError, "k shape", x[:, :1], x, c, slots),
        (ValueError, "k shape", x[..., :56], x, c, slots),
        (ValueError, "v shape", x, x[:2], c, slots),
        (TypeError, "k must be torch.float16", x.bfloat16(), x, c, slots),
        (TypeError, "v must be torch.float16", x, x.bfloat16(), c, slots),
        (TypeError, "v must be torch.bfloat16", x.bfloat16(), x, f8, slots),
        (TypeError, "k must be fp16 or bf16", x.float(), x.float(), f8, slots),
        (ValueError, "slots shape", x, x, c, slots[:2]),
        (ValueError, "slots shape", x, x, c, slots[:, None]),
        (TypeError, "slots must be torch.int64", x, x, c, slots.int()),
    ]:
        with pytest.raises(error, match=match):
            ops.kv_cache_write(k, v, *cache, s)
        with pytest.raises(error, match=match):
            ops.rope_kv_cache_write(q, k, v, table, slots, *cache, s)
    for error, match, qq, t, p in [
        (ValueError, "q must be", q[0], table, slots),
        (ValueError, "q must be", q[:, :0], table, slots),
        (ValueError, "q shape", q[:2], table, slots),
        (ValueError, "q shape", q[..., :8], table, slots),
        (TypeError, "q must be torch.float16", q.bfloat16(), table, slots),
        (ValueError, "cos_sin must be", q, table[0], slots),
        (ValueError, "cos_sin must be", q, table[:0], slots),
        (TypeError, "cos_sin must be fp32", q, table.half(), slots),
        (ValueError, "even, above 0", q, table[:, :31], slots),
        (ValueError, "even, above 0", q, table[:, :0], slots),
        (ValueError, "even, above 0", q, torch.zeros((9, 66)), slots),
        (ValueError, "positions shape", q, table, slots[:1]),
        (TypeError, "positions must be torch.int64", q, table, slots.int()),
    ]:
        with pytest.raises(error, match=match):
            ops.rope_kv_cache_write(qq, x, x, t, p, *c, slots)


def test_reads_and_attention_are_refused() -> None:
    c = (torch.zeros((2, 2, 16, 64), dtype=torch.float16), torch.zeros((2, 2, 16, 64), dtype=torch.float16), None, None)
    f8 = (c[0].to(kc.F8), c[1].to(kc.F8), torch.ones((2, 2, 16)), torch.ones((2, 2, 16)))
    slots = torch.arange(3)
    with pytest.raises(TypeError, match="out_dtype must be torch.float16 like"):
        ops.kv_cache_read(*c, slots, torch.bfloat16)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.kv_cache_read(*f8, slots, torch.float32)
    with pytest.raises(ValueError, match="slots shape"):
        ops.kv_cache_read(*c, slots[None], torch.float16)
    with pytest.raises(TypeError, match="slots must be"):
        ops.kv_cache_read(*c, slots.int(), torch.float16)
    q, t, n = torch.zeros((3, 4, 64), dtype=torch.float16), torch.zeros((3, 2), dtype=torch.int32), slots.int()
    for error, match, args in [
        (ValueError, "q must be", (q[0], *c, t, n, 1.0)),
        (ValueError, "a multiple of 2 heads", (q[:, :3], *c, t, n, 1.0)),
        (ValueError, "a multiple of 2 heads", (q[:, :0], *c, t, n, 1.0)),
        (ValueError, "q shape", (q[..., :56], *c, t, n, 1.0)),
        (TypeError, "q must be torch.float16", (q.bfloat16(), *c, t, n, 1.0)),
        (TypeError, "q must be fp16 or bf16", (q.float(), *f8, t, n, 1.0)),
        (ValueError, "block_table must be", (q, *c, t[0], n, 1.0)),
        (ValueError, "block_table must be", (q, *c, t[:2], n, 1.0)),
        (TypeError, "block_table must be", (q, *c, t.long(), n, 1.0)),
        (ValueError, "seq_lens shape", (q, *c, t, n[:2], 1.0)),
        (TypeError, "seq_lens must be", (q, *c, t, n.long(), 1.0)),
        (ValueError, "window", (q, *c, t, n, 1.0, -1)),
        (ValueError, "too large", (q, *c, t[:, :1].expand(3, 1 << 27), n, 1.0)),
        (ValueError, "too large", (q[:1].expand(1 << 21, -1, -1), *c, t[:1].expand(1 << 21, -1),
                                   n[:1].expand(1 << 21), 1.0)),
    ]:
        with pytest.raises(error, match=match):
            ops.paged_attention(*args)


def _c_cache(**changed):  # type: ignore[no-untyped-def]
    """A cache of addresses that are never read: every call below is refused on the host."""
    three = ctypes.c_int64 * 3
    fields = {"k": 0x10000, "v": 0x20000, "k_scale": 0x30000, "v_scale": 0x40000, "pages": 4, "heads": 2,
              "page_size": 16, "head_dim": 64, "dtype": 0, "k_strides": three(2048, 1024, 64),
              "v_strides": three(2048, 1024, 64), "k_scale_strides": three(32, 16, 1),
              "v_scale_strides": three(32, 16, 1)}
    fields.update(changed)
    return ctypes.byref(_lib.TfKvCache(**fields))


BAD_CACHES = [
    ({"dtype": 1}, b"neither"), ({"dtype": 3}, b"neither"), ({"k": None}, b"null"), ({"v": None}, b"null"),
    ({"pages": 0}, b"above 0"), ({"heads": -1}, b"above 0"), ({"page_size": 0}, b"above 0"), ({"heads": 70000}, b"65535"),
    ({"pages": (1 << 31) + 1}, b"2^31"), ({"page_size": (1 << 24) + 1}, b"2^24"), ({"head_dim": 60}, b"head_dim"),
    ({"head_dim": 264}, b"head_dim"), ({"head_dim": 0}, b"head_dim"), ({"k": 0x10008}, b"unaligned"),
    ({"v_strides": (ctypes.c_int64 * 3)(2048, 1024, 60)}, b"unaligned"),
    ({"v_strides": (ctypes.c_int64 * 3)(2048, -1024, 64)}, b"negative"),
    ({"k_strides": (ctypes.c_int64 * 3)(2048, 1024, 1 << 24)}, b"apart"),
    ({"dtype": 2, "k_scale": None}, b"null"), ({"dtype": 2, "v_scale_strides": (ctypes.c_int64 * 3)(1, 1, -1)}, b"negative"),
    ({"dtype": 2, "k_scale_strides": (ctypes.c_int64 * 3)(1, 1, 1 << 24)}, b"apart"),
]


def test_c_entries_refuse_before_any_launch() -> None:
    h = _lib.lib()
    x, i = 0x50000, 0x60000

    def write(c, k=x, kt=128, kh=64, dtype=0, slots=i, t=1):  # type: ignore[no-untyped-def]
        return h.tf_kv_cache_write(c, k, kt, kh, x, 128, 64, dtype, slots, t, None)

    def rope(c, q=x, heads=4, cs=x, far=9, rot=64, out=x, t=1, pos=i):  # type: ignore[no-untyped-def]
        return h.tf_rope_kv_cache_write(c, q, 256, 64, heads, x, 128, 64, x, 128, 64, 0, cs, far, rot, 0, pos, i, out, t, None)

    def read(c, out=x, slots=i, t=1, dtype=0):  # type: ignore[no-untyped-def]
        return h.tf_kv_cache_read(c, slots, out, x, dtype, t, None)

    def attend(c, q=x, qr=256, heads=4, dtype=0, table=i, width=4, m=2, window=0, ws=x, size=1 << 30, lens=i, stride=4):  # type: ignore[no-untyped-def]
        return h.tf_paged_attention(c, q, qr, 64, heads, dtype, table, stride, width, lens, m, 1.0, window, x, ws, size, None)

    for changed, message in BAD_CACHES:
        for call in (write, rope, read, attend):
            assert call(_c_cache(**changed)) == _lib.TF_EINVAL
            assert message in h.tf_last_error(), (changed, h.tf_last_error())
    ok = _c_cache()
    for bad, message in [({"v": 0x10000}, b"one place"), ({"dtype": 2, "v_scale": 0x30000}, b"scales of keys")]:
        for call in (write, rope):
            assert call(_c_cache(**bad)) == _lib.TF_EINVAL and message in h.tf_last_error()
    for call, changed, message in [
        (write, {"k": None}, b"null"), (write, {"k": x + 2}, b"aligned"), (write, {"kt": 129}, b"aligned"),
        (write, {"kh": 4}, b"aligned"), (write, {"dtype": 2}, b"unknown dtype"), (write, {"slots": None}, b"null"),
        (write, {"t": -1}, b"t >= 0"),
        (rope, {"q": None}, b"null"), (rope, {"heads": 0}, b"q_heads"), (rope, {"heads": 70000}, b"q_heads"),
        (rope, {"cs": None}, b"null"), (rope, {"cs": x + 4}, b"aligned"), (rope, {"far": 0}, b"max_positions"),
        (rope, {"rot": 66}, b"rot"), (rope, {"rot": 3}, b"rot"), (rope, {"rot": 0}, b"rot"), (rope, {"out": x + 8}, b"aligned"),
        (rope, {"pos": None}, b"null"), (rope, {"t": -1}, b"t >= 0"),
        (read, {"out": None}, b"null"), (read, {"slots": None}, b"null"), (read, {"t": -1}, b"t >= 0"),
        (read, {"dtype": 7}, b"unknown dtype"),
        (attend, {"q": None}, b"null"), (attend, {"q": x + 8}, b"aligned"), (attend, {"qr": 4}, b"aligned"),
        (attend, {"heads": 3}, b"multiple"), (attend, {"heads": 0}, b"multiple"), (attend, {"table": None}, b"null"),
        (attend, {"lens": None}, b"null"), (attend, {"width": -1}, b"size"), (attend, {"m": -1}, b"size"),
        (attend, {"width": 1 << 27}, b"2^31"), (attend, {"width": 1 << 62}, b"2^31"),
        (attend, {"m": 1 << 22}, b"2^31"), (attend, {"window": -1}, b"window"), (attend, {"ws": None, "width": 4000}, b"workspace"),
        (attend, {"ws": x + 4, "width": 4000}, b"16-byte"), (attend, {"size": 64, "width": 4000}, b"workspace too small"), (attend, {"stride": -4}, b"negative"),
    ]:
        assert call(ok, **changed) == _lib.TF_EINVAL
        assert message in h.tf_last_error(), (call.__name__, changed, h.tf_last_error())
    assert write(ok, t=0) == rope(ok, t=0) == read(ok, t=0) == attend(ok, m=0) == _lib.TF_OK
    assert write(None) == rope(None) == read(None) == attend(None) == _lib.TF_EINVAL
    need = h.tf_paged_attention_workspace_bytes
    assert need(ok, 2, 4, 4000, 0) > 0 and need(ok, 2, 4, 4000, 100) == need(ok, 2, 4, 1, 0) == need(ok, 0, 4, 40, 0) == 0
    assert need(ok, 2, 3, 4, 0) == need(None, 2, 4, 4, 0) == need(ok, 2, 4, 1 << 40, 0) == need(ok, 2, 4, 4, -1) == -1
    assert need(ok, -1, 4, 4, 0) == need(ok, 1 << 40, 4, 4, 0) == need(_c_cache(head_dim=4), 2, 4, 4, 0) == -1


def test_page_division_is_exact() -> None:
    """n / d as (n * mul) >> (31 + shift), mul = ceil(2^(31 + shift) / d), for every page size's multiples and their
    neighbours up to 2^31 and for numbers in between."""
    rng = np.random.default_rng(0)
    for d in [*range(1, 300), 1000, 4097, 65535, 65536, (1 << 24) - 1, 1 << 24]:
        shift = (d - 1).bit_length()
        mul = -(-(1 << (31 + shift)) // d)
        assert mul < 1 << 32
        top = ((1 << 31) - 1) // d * d
        some = [int(x) for x in rng.integers(0, 1 << 31, 200)] + [0, 1, top - 1, top, (1 << 31) - 1]
        some += [int(x) // d * d + e for x in rng.integers(d + 1, 1 << 30, 100) for e in (-1, 0, 1)]
        assert all(n * mul >> (31 + shift) == n // d for n in some)


def test_kernel_limits_match_the_library() -> None:
    header = (_lib.LIB_PATH.parents[2] / "include" / "tokenforge_hip.h").read_text()
    assert f"#define TF_KV_MAX_HEAD_DIM {kv.MAX_HEAD_DIM}" in header
    assert f"#define TF_DTYPE_E4M3 {_lib.DTYPE_E4M3}" in header


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_the_attentions_bound_sees_a_token(dtype: torch.dtype) -> None:
    """What the bound is held to: an oracle that misses one token, reads another page, has the window off by one or the
    scale by 2% is outside it."""
    lens = [60]
    table, pages = kc.tables(lens, 16)
    c = kc.cache(pages, 1, 16, 64, dtype, False)
    q = _rows(1, 2, 64, dtype, 0)
    out = ops.paged_attention(q, *c.to("cpu"), table, torch.tensor(lens, dtype=torch.int32), 0.05, 20)
    kc.check_attention(out, q, c, table, lens, 0.05, 20)
    swapped = table.clone()
    swapped[0, 3] = table[0, 2]
    for t, n, scale, window in ((table, 59, 0.05, 20), (swapped, 60, 0.05, 20), (table, 60, 0.05, 21), (table, 60, 0.051, 20)):
        with pytest.raises(AssertionError):
            kc.check_attention(out, q, c, t, [n], scale, window)
