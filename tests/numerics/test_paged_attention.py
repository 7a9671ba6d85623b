"""The paged attention on the GPU against its definition in 64 bits, at the lengths, pages, heads, layouts and values
where it can go wrong. Bounds: ``kv_cases.check_attention``."""

from __future__ import annotations

import random

import pytest
import torch
from torch.library import opcheck

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import kv_cases as kc

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp16-e4m3", "bf16-e4m3"]


def _queries(m: int, q_heads: int, d: int, dtype: torch.dtype, seed: int = 0) -> torch.Tensor:
    q = torch.randn((m, q_heads, d), generator=kc.gen("q", m, q_heads, d, seed))
    q[..., :: max(1, d // 4)] *= 2.0
    return q.to(dtype)


LINE = 1 << 15  # tokens of a table's row from which items share workgroups, whatever the sequences' lengths


def _run(device, lens, heads, group, d, page, dtype, fp8, window=0, width=None, tokens_first=False, scale=None, seed=0):  # type: ignore[no-untyped-def]
    table, pages = kc.tables(lens, page, width, seed)
    c = kc.cache(pages, heads, page, d, dtype, fp8, seed, tokens_first)
    q = _queries(len(lens), heads * group, d, dtype, seed)
    scale = d**-0.5 if scale is None else scale
    out = ops.paged_attention(q.to(device), *c.to(device), table.to(device),
                              torch.tensor(lens, dtype=torch.int32, device=device), scale, window)
    assert out.shape == q.shape and out.dtype == dtype
    kc.check_attention(out, q, c, table, lens, scale, window)
    return out


LENS = [[1], [0], [16], [17], [33, 0, 64, 65, 1], [300, 5, 129, 0], [1500], [700, 2, 31]]


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("capacity", [0, LINE])
def test_lengths(capacity: int, d: int, lens: list[int], dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, lens, 2, 7, d, 16, dtype, fp8, width=capacity // 16)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("page", [1, 5, 8, 24, 32, 48, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_page_sizes(d: int, page: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, [200, 1, 77], 2, 4, d, page, dtype, fp8)
    _run(device, [200, 1, 77], 2, 4, d, page, dtype, fp8, width=LINE // page)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("d", [8, 40, 72, 80, 96, 112, 136, 192, 248])
@pytest.mark.parametrize("page", [16, 24])
def test_odd_head_lengths(page: int, d: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, [150, 31, 400], 3, 2, d, page, dtype, fp8)
    _run(device, [150, 31, 400], 3, 2, d, page, dtype, fp8, width=LINE // page)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize(("heads", "group"), [(1, 1), (12, 1), (1, 16), (2, 17), (1, 71), (5, 3)])
def test_head_layouts(heads: int, group: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, [333, 40], heads, group, 128, 16, dtype, fp8)
    _run(device, [333, 40], heads, group, 128, 16, dtype, fp8, width=LINE // 16)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("window", [1, 15, 16, 64, 100, 5000])
@pytest.mark.parametrize("page", [16, 24])
def test_windows(page: int, window: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, [400, 99, 16, 0, 1], 2, 4, 128, page, dtype, fp8, window=window)
    _run(device, [9000, 99, 16, 0, 1], 2, 4, 128, page, dtype, fp8, window=12 * window)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
def test_long_sequences_and_large_batches(d: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    _run(device, [9001, 3], 2, 7, d, 16, dtype, fp8)
    # more sequences than a workgroup has threads, and than the grid has workgroups; empty ones at both ends
    lens = [0, 0] + [(37 * i) % 91 for i in range(598)] + [0]
    _run(device, lens, 1, 2, d, 16, dtype, fp8, width=40)
    _run(device, lens, 1, 2, d, 16, dtype, fp8, width=LINE // 16)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[180000, 0, 90000], [1000] * 100, [5000, 70, 9000, 3, 33, 12000] * 3], ids=["2", "100", "18"])
def test_every_way_to_share_the_work(lens: list[int], fp8: bool, device: torch.device) -> None:
    """Parts of 4 to 32 steps an item, and parts that begin and end inside items, of many lengths."""
    for d in (64, 136):
        _run(device, lens, 1 if len(lens) < 10 else 3, 3, d, 64, torch.bfloat16, fp8, width=180000 // 64 + 1)
        _run(device, lens[:1] + lens[-1:], 1, 3, d, 64, torch.bfloat16, fp8)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize(("d", "group"), [(64, 4), (64, 20), (128, 4), (128, 20), (256, 4)])
@pytest.mark.parametrize("whole", [False, True], ids=["shared", "whole"])
def test_calls_of_many_bytes(whole: bool, d: int, group: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Below and past 100 MiB of keys and values on the line, and 384 MiB in the table of items that a workgroup takes
    whole: the same four sequences again and again, over the same pages."""
    row = 2 * d * (1 if fp8 else 2)
    capacity = (512 << 10) // row if whole else LINE
    lens = [min(2049, capacity), capacity // 2 + 1 if whole else 1777, 1, 300]
    past = 101 if whole else (60 << 20) // (sum(lens) * row) + 1  # 808 items of 512 KB; 120 MiB of 2 heads
    table, pages = kc.tables(lens, 16, capacity // 16)
    c = kc.cache(pages, 2, 16, d, dtype, fp8)
    q = _queries(len(lens), 2 * group, d, dtype)
    for n in (80 if whole else past // 4, past):
        out = ops.paged_attention(q.repeat(n, 1, 1).to(device), *c.to(device), table.repeat(n, 1).to(device),
                                  torch.tensor(lens * n, dtype=torch.int32, device=device), d**-0.5, 0)
        for at in (0, n // 2, n - 1):
            kc.check_attention(out[4 * at:4 * at + 4], q, c, table, lens, d**-0.5)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("capacity", [0, LINE])
def test_layouts(capacity: int, page: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Caches laid out by token, keys and values in one tensor, strided queries, tables, lengths: the results of
    contiguous copies, bit for bit."""
    lens, heads, group, d = [210, 64, 0, 700], 2, 4, 128
    table, pages = kc.tables(lens, page, capacity // page)
    c = kc.cache(pages, heads, page, d, dtype, fp8)
    q = _queries(4, heads * group, d, dtype).to(device)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    t = table.to(device)
    k, v, ks, vs = c.to(device)
    want = ops.paged_attention(q, k, v, ks, vs, t, n, 0.1, 0)
    kc.check_attention(want, q.cpu(), c, table, lens, 0.1)

    def same(*args):  # type: ignore[no-untyped-def]
        assert torch.equal(ops.paged_attention(*args, 0.1, 0), want)

    c.tokens_first = True
    same(q, *c.to(device), t, n)
    both = torch.stack([k.view(torch.uint8), v.view(torch.uint8)], 3).view(k.dtype)  # [pages, heads, page, 2, d]
    same(q, both[..., 0, :], both[..., 1, :], ks, vs, t, n)
    wide = torch.zeros((pages, heads, page, d + 24), dtype=torch.uint8 if fp8 else dtype, device=device)
    wide[..., 8:d + 8] = k.view(torch.uint8) if fp8 else k
    same(q, wide[..., 8:d + 8].view(k.dtype) if fp8 else wide[..., 8:d + 8], v, ks, vs, t, n)
    joined = torch.randn((4, 3000), device=device).to(dtype)
    joined[:, 8:8 + q[0].numel()] = q.flatten(1)
    same(joined[:, 8:8 + q[0].numel()].unflatten(1, (-1, d)), k, v, ks, vs, t, n)
    odd = torch.zeros((4, heads * group, d + 3), dtype=dtype, device=device)
    odd[..., 3:] = q
    same(odd[..., 3:], k, v, ks, vs, t, n)
    same(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, ks, vs, t, n)
    same(q, k, v, ks, vs, torch.cat([t, t + 100000], 1)[:, : t.shape[1]], n)
    same(q, k, v, ks, vs, t.t().contiguous().t(), n.repeat_interleave(2)[::2])


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("capacity", [0, LINE])
def test_nothing_outside_a_sequence_takes_part(capacity: int, d: int, page: int, dtype: torch.dtype, fp8: bool,
                                               device: torch.device) -> None:
    """NaN and infinities behind the last token, before the window and in every other page; entries of the table
    behind the last page that lead nowhere; lengths beyond the table and below zero."""
    lens, window = [77, 1, 130, 0, 250], 60
    table, pages = kc.tables(lens, page, capacity // page)
    c = kc.cache(pages, 2, page, d, dtype, fp8)
    q = _queries(5, 4, d, dtype)
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(max(0, n - window), n):
            used[table[b, i // page], i % page] = True
    for x in (c.k, c.v):
        bits = x.view(torch.uint8 if fp8 else torch.int16)
        bad = {torch.float16: (0x7E00, -0x0400), torch.bfloat16: (0x7FC0, -0x0080)}.get(x.dtype, (0x7F, 0xFF))
        fill = torch.where(torch.arange(d) % 2 == 0, bad[0], bad[1]).to(bits.dtype)  # NaN and -infinity (e4m3: NaN)
        bits.copy_(torch.where(used[:, None, :, None], bits, fill))
    if fp8:
        for s in (c.ks, c.vs):
            s.copy_(torch.where(used[:, None], s, float("inf")))
    wild = table.clone()
    for b, n in enumerate(lens):
        wild[b, -(-n // page):] = torch.tensor([2**31 - 1, -(2**31), pages, -1] * LINE)[: wild.shape[1] - -(-n // page)]
    out = ops.paged_attention(q.to(device), *c.to(device), wild.to(device),
                              torch.tensor(lens, dtype=torch.int32, device=device), d**-0.5, window)
    for x in (c.k, c.v):  # finite for the oracle, which multiplies them by nothing
        bits = x.view(torch.uint8 if fp8 else torch.int16)
        bits.copy_(torch.where(used[:, None, :, None], bits, torch.zeros_like(bits)))
    kc.check_attention(out, q, c, table, lens, d**-0.5, window)
    if capacity:
        return
    # lengths past the table end with it, lengths below zero are none
    far = torch.tensor([2**31 - 1, -5, 130, -(2**31), 250], dtype=torch.int32, device=device)
    c = kc.cache(pages, 2, page, d, dtype, fp8)
    out = ops.paged_attention(q.to(device), *c.to(device), table.clamp(min=0).to(device), far, d**-0.5, 0)
    kc.check_attention(out, q, c, table.clamp(min=0), [table.shape[1] * page, 0, 130, 0, 250], d**-0.5)


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("capacity", [0, LINE])
def test_pages_that_are_not_there(capacity: int, page: int, dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Page numbers outside the cache inside a sequence: their tokens take no part; a sequence of such pages alone
    gives zeros."""
    lens = [200, 90, 48]
    table, pages = kc.tables(lens, page, capacity // page)
    table[0, 1], table[0, 3], table[1, 0] = -1, pages, 2**31 - 1
    table[2] = -7
    c = kc.cache(pages, 2, page, 128, dtype, fp8)
    q = _queries(3, 6, 128, dtype)
    out = ops.paged_attention(q.to(device), *c.to(device), table.to(device),
                              torch.tensor(lens, dtype=torch.int32, device=device), 0.1, 0)
    kc.check_attention(out, q, c, table, lens, 0.1)
    assert not out[2].any()


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
def test_infinite_and_nan_values_that_take_part(dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """As the softmax's expression gives them: an infinite value in its channel alone, a NaN key in its heads, a key
    that scores -infinity not at all."""
    lens = [100, 3000]
    table, pages = kc.tables(lens, 16)
    c = kc.cache(pages, 2, 16, 128, dtype, fp8)
    q = torch.ones((2, 4, 128), dtype=dtype)
    k, v, ks, vs = c.to(device)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    t = table.to(device)
    base = ops.paged_attention(q.to(device), k, v, ks, vs, t, n, 0.001, 0)
    if not fp8:
        v2 = v.clone()
        v2[table[1, 20], 1, 3, 5] = float("inf")
        v2[table[1, 60], 0, 3, 7] = float("-inf")
        out = ops.paged_attention(q.to(device), k, v2, ks, vs, t, n, 0.001, 0)
        assert (out[1, 2:, 5] == float("inf")).all() and (out[1, :2, 7] == float("-inf")).all()
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1, 2:, 5] = keep[1, :2, 7] = False
        assert torch.equal(out[keep], base[keep])
        k2 = k.clone()
        k2[table[0, 2], 0, 3] = float("-inf")
        out = ops.paged_attention(q.to(device), k2, v, ks, vs, t, n, 0.001, 0)
        gone = kc.Cache(c.k, c.v, None, None)
        assert torch.isfinite(out).all() and torch.equal(out[1], base[1]) and torch.equal(out[0, 2:], base[0, 2:])
        one = torch.cat([torch.arange(35), torch.arange(36, 100)])
        from oracle import kv_cache as okv

        kv = [okv.tokens(kc.values(x), None, table[0].numpy(), 0, 100)[one.numpy()] for x in (gone.k, gone.v)]
        want, size, _ = okv.attention(kc.values(q[0]), *kv, 0.001)
        assert (abs(kc.values(out[0, :2]) - want[:2]) <= 2 * kc.EPS[dtype] * size[:2]).all()
    k2 = k.clone()
    k2.view(torch.uint8 if fp8 else dtype)[table[1, 30], 1, 2, 9] = 0x7F if fp8 else float("nan")
    out = ops.paged_attention(q.to(device), k2, v, ks, vs, t, n, 0.001, 0)
    assert torch.isnan(out[1, 2:]).all() and torch.equal(out[1, :2], base[1, :2]) and torch.equal(out[0], base[0])


@pytest.mark.parametrize(("dtype", "fp8"), TYPES, ids=IDS)
def test_scores_of_any_size(dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Scales that make one token take all, that turn the order round, and none at all (the mean)."""
    for scale in (30.0, -1.0, 0.0, 1e-6):
        _run(device, [400, 37], 2, 2, 128, 16, dtype, fp8, scale=scale)


def test_scales_far_apart(device: torch.device) -> None:
    """e4m3 scales over 60 binary orders, in keys and values: no probability times a scale is cut at the type's end."""
    lens = [300, 20]
    table, pages = kc.tables(lens, 16)
    for dtype in (torch.float16, torch.bfloat16):
        c = kc.cache(pages, 2, 16, 128, dtype, True)
        c.vs *= torch.exp2(torch.randint(-40, 3, c.vs.shape, generator=kc.gen("far")).float())
        c.ks *= torch.exp2(torch.randint(-40, 1, c.ks.shape, generator=kc.gen("far2")).float())
        c.vs[:, 1] *= -1.0  # no quantizer writes such; they multiply all the same
        c.ks[:, 1] *= -1.0
        q = _queries(2, 4, 128, dtype)
        out = ops.paged_attention(q.to(device), *c.to(device), table.to(device),
                                  torch.tensor(lens, dtype=torch.int32, device=device), 0.1, 0)
        kc.check_attention(out, q, c, table, lens, 0.1)


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_past_32_bits(fp8: bool, device: torch.device) -> None:
    """Pages whose byte and element offsets pass 2^32, page by page and head by head."""
    dtype, page, d, lens = torch.bfloat16, 16, 128, [100, 40]
    table, pages = kc.tables(lens, page, spare=0)
    c = kc.cache(pages, 2, page, d, dtype, fp8)
    q = _queries(2, 8, d, dtype)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    far = (1 << 32) // (2 * page * d) + 5  # pages up to 2^32 elements
    for heads_first in (False, True):
        dev = []
        for t, tail in ((c.k, (page, d)), (c.v, (page, d)), (c.ks, (page,)), (c.vs, (page,))):
            if t is None:
                dev.append(None)
                continue
            shape = (2, far + pages, *tail) if heads_first else (far + pages, 2, *tail)
            big = torch.empty(shape, dtype=t.dtype, device=device)
            big = big.transpose(0, 1) if heads_first else big
            big[far:] = t.to(device)
            dev.append(big)
        out = ops.paged_attention(q.to(device), *dev, (table + far * (table >= 0)).to(torch.int32).to(device), n, 0.1, 0)
        kc.check_attention(out, q, c, table, lens, 0.1)
        del big, dev
        torch.cuda.empty_cache()


@pytest.mark.parametrize("fp8", [False, True])
def test_graph_replays_follow_lengths_and_tables(fp8: bool, device: torch.device) -> None:
    """Two captured graphs and eager calls in turn: each replay equals the eager call on what the buffers hold."""
    dtype, page, lens = torch.bfloat16, 16, [800, 3, 120]
    table, pages = kc.tables([1024, 1024, 1024], page)
    c = kc.cache(pages, 2, page, 128, dtype, fp8)
    args = c.to(device)
    q, t = _queries(3, 14, 128, dtype).to(device), table.to(device)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    q2 = _queries(3, 14, 128, dtype, 1).to(device)
    ops.paged_attention(q, *args, t, n, 0.1, 0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for query, window in ((q, 0), (q2, 100)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(query, *args, t, n, 0.1, window))
        graphs.append(g)
    for step in range(4):
        n.copy_(torch.tensor([800 + step, 0 if step == 2 else 3 + 300 * step, 120 + 7 * step], dtype=torch.int32))
        if step == 3:
            t.copy_(t.flip(0))
        graphs[0].replay()
        graphs[1].replay()
        graphs[0].replay()
        want = [ops.paged_attention(query, *args, t, n, 0.1, w) for query, w in ((q, 0), (q2, 100))]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    kc.check_attention(outs[0], q.cpu(), c, t.cpu(), n.cpu().tolist(), 0.1)


def test_two_streams_and_repeats(device: torch.device) -> None:
    lens = [2500, 30, 900]
    table, pages = kc.tables(lens, 16)
    c = kc.cache(pages, 4, 16, 128, torch.bfloat16, True)
    args, t = c.to(device), table.to(device)
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    qs = [_queries(3, 28, 128, torch.bfloat16, i).to(device) for i in range(2)]
    want = [ops.paged_attention(q, *args, t, n, 0.1, 0) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(qs[i], *args, t, n, 0.1, 0))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_opcheck_and_compile(device: torch.device) -> None:
    table, pages = kc.tables([40, 9], 16)
    c = kc.cache(pages, 2, 16, 64, torch.float16, True).to(device)
    q = _queries(2, 4, 64, torch.float16).to(device)
    args = (q, *c, table.to(device), torch.tensor([40, 9], dtype=torch.int32, device=device), 0.125, 0)
    opcheck(ops.paged_attention, args, test_utils=("test_faketensor", "test_aot_dispatch_dynamic"))
    c16 = kc.cache(pages, 2, 16, 64, torch.float16, False).to(device)
    opcheck(ops.paged_attention, (q, *c16, *args[5:]))  # test_schema multiplies its inputs, which e4m3 lacks
    got = torch.compile(lambda *a: ops.paged_attention(*a) * 2, fullgraph=True, backend="aot_eager")(*args)
    assert torch.equal(got, ops.paged_attention(*args) * 2)
    assert ops.paged_attention(q[:0], *c, table[:0].to(device), args[6][:0], 0.125, 0).shape == (0, 4, 64)
    assert not ops.paged_attention(q, *c, table[:, :0].to(device), args[6], 0.125, 0).any()


@pytest.mark.parametrize("seed", range(24))
def test_drawn_calls(seed: int, device: torch.device) -> None:
    """Calls of no pattern: every combination of sizes, layouts and types that the operator takes can come up."""
    rng = random.Random(seed)
    dtype, fp8 = rng.choice(TYPES)
    page = rng.choice((16, 16, 32, 64, rng.randint(1, 70)))
    heads, group = rng.choice((1, 2, 3, 8)), rng.choice((1, 2, 7, 15, 16, 17, 31, 33, 40))
    d = rng.choice((64, 128, 256, 8 * rng.randint(1, 32)))
    longest = rng.choice((20, 100, 700, 4000))
    lens = [rng.choice((0, 1, rng.randint(1, longest), rng.randint(1, longest))) for _ in range(rng.choice((1, 3, 20, 70)))]
    width = rng.choice((0, 0, LINE // page, rng.randint(1, 2 * longest) // page))
    _run(device, lens, heads, group, d, page, dtype, fp8, window=rng.choice((0, 0, rng.randint(1, longest))), width=width,
         tokens_first=rng.random() < 0.3, scale=rng.choice((None, None, rng.uniform(-0.5, 0.5))), seed=seed)
