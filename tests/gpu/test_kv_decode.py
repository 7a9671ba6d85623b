"""The cache's operators and the attention as a decoder uses them together: a prompt written and read back, decode steps
that each write their tokens and attend over all of them, and FP8 layers with them in a captured graph."""

from __future__ import annotations

import pytest
import torch

import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)
from tests.numerics import kv_cases as kc

pytestmark = pytest.mark.gpu
ops = torch.ops.tokenforge
EPS = 1e-6


def _table(rot: int, far: int, device: torch.device) -> torch.Tensor:
    freq = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(far, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


@pytest.mark.parametrize(("dtype", "fp8"), [(torch.float16, False), (torch.bfloat16, True)], ids=["fp16", "bf16-e4m3"])
def test_prompt_then_decode_steps(dtype: torch.dtype, fp8: bool, device: torch.device) -> None:
    """Three conversations of 14 query and 2 key-value heads of 64: prompts of 70, 1 and 16 tokens, then 20 steps."""
    q_heads, heads, d, page, steps = 14, 2, 64, 16, 20
    prompts = [70, 1, 16]
    table, pages = kc.tables([n + steps for n in prompts], page)
    c = kc.cache(pages, heads, page, d, dtype, fp8)
    cache = c.to(device)
    angles = _table(d, 256, device)
    width = (q_heads + 2 * heads) * d
    g = kc.gen("decode")

    def slots_of(b: int, at: torch.Tensor) -> torch.Tensor:
        return table[b, at // page].long() * page + at % page

    def qkv(t: int) -> list[torch.Tensor]:
        x = torch.randn((t, width), generator=g).to(dtype).to(device)
        return [p.unflatten(1, (-1, d)) for p in x.split((q_heads * d, heads * d, heads * d), 1)]

    positions = torch.cat([torch.arange(n) for n in prompts])
    slots = torch.cat([slots_of(b, torch.arange(n)) for b, n in enumerate(prompts)])
    q, k, v = qkv(sum(prompts))
    q = ops.rope_kv_cache_write(q, k, v, angles, positions.to(device), *cache, slots.to(device), False)
    # read back: the values as they were written, keys turned (e4m3: within half a code of the row's largest)
    kb, vb = ops.kv_cache_read(*cache, slots.to(device), dtype)
    if fp8:
        top = v.float().abs().amax(-1, keepdim=True)
        assert ((vb.float() - v.float()).abs() <= top * 2.0**-4 * (1 + 2.0**-7)).all()
    else:
        assert torch.equal(vb, v)
    norms = [x.float().square().sum(-1).sqrt() for x in (kb, k)]
    assert ((norms[0] - norms[1]).abs() <= norms[1] * (2.0**-4 if fp8 else 2.0**-9)).all()

    lens = list(prompts)
    for _ in range(steps):
        q, k, v = qkv(3)
        at = torch.tensor(lens)
        slots = torch.stack([slots_of(b, at[b]) for b in range(3)]).to(device)
        q = ops.rope_kv_cache_write(q, k, v, angles, at.to(device), *cache, slots, False)
        lens = [n + 1 for n in lens]
        out = ops.paged_attention(q, *cache, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device),
                                  d**-0.5)
        now = kc.Cache(*(None if x is None else x.cpu() for x in cache))
        kc.check_attention(out, q.cpu(), now, table, lens, d**-0.5)
    # one token's attention over a prefix that was read back, by torch in 64 bits
    at = torch.arange(lens[0])
    kb, vb = (x.double().transpose(0, 1) for x in ops.kv_cache_read(*cache, slots_of(0, at).to(device), dtype))
    p = torch.softmax(q[0].double().unflatten(0, (heads, -1)) @ kb.transpose(1, 2).contiguous() * d**-0.5, -1)
    want = (p @ vb.contiguous()).flatten(0, 1)
    size = (p @ vb.abs().contiguous()).flatten(0, 1)
    # e4m3 values were rounded to 16 bits on their way back: half a step of each, in the scores (at most 4 in size here
    # times 64 products) and in the values
    err = (kc.EPS[dtype] * 2 + (kc.EPS[dtype] * 16 if fp8 else 0)) * size + 2.0**-12 * size
    assert ((out[0].double() - want).abs() <= err).all()


H, Q_HEADS, KV_HEADS, D, INTER = 896, 14, 2, 64, 4864


def _layers(count: int, device: torch.device) -> list[dict[str, torch.Tensor]]:
    out = []
    for i in range(count):
        g = torch.Generator(device=device).manual_seed(i)
        layer = {}
        for name, n, k in (("qkv", H + 2 * KV_HEADS * D, H), ("o", H, H), ("gate_up", 2 * INTER, H), ("down", H, INTER)):
            w = torch.randn((n, k), generator=g, device=device) * 100
            layer[name] = w.clamp(-448, 448).to(torch.float8_e4m3fn)
            layer[name + "_scale"] = torch.full((-(-n // 128), -(-k // 128)), 0.01 / k**0.5, device=device)
        layer["bias"] = torch.randn(H + 2 * KV_HEADS * D, generator=g, device=device).bfloat16()
        layer["norm1"], layer["norm2"] = (torch.ones(H, dtype=torch.bfloat16, device=device) for _ in range(2))
        out.append(layer)
    return out


def _step(x, layers, caches, angles, positions, slots, table, lens):  # type: ignore[no-untyped-def]
    """A decode step through FP8 layers: every linear on codes with a scale per 128."""
    hidden = None
    m = x.shape[0]

    def linear(q, s, layer, name, bias=None):  # type: ignore[no-untyped-def]
        return ops.fp8_block_linear(q, s, layer[name], layer[name + "_scale"], bias, torch.bfloat16, "hip")

    for layer, cache in zip(layers, caches):
        q, s, h = ops.add_rmsnorm_fp8_quant(x, hidden, layer["norm1"], EPS, 128)
        hidden = x if hidden is None else h
        y = linear(q, s, layer, "qkv", layer["bias"])
        parts = [p.unflatten(1, (-1, D)) for p in y.split((H, KV_HEADS * D, KV_HEADS * D), 1)]
        qr = ops.rope_kv_cache_write(*parts, angles, positions, *cache, slots, False)
        a = ops.paged_attention(qr, *cache, table, lens, D**-0.5)
        x = linear(*ops.fp8_quant(a.reshape(m, H), 128), layer, "o")
        q, s, hidden = ops.add_rmsnorm_fp8_quant(x, hidden, layer["norm2"], EPS, 128)
        x = linear(*ops.silu_mul_fp8_quant(linear(q, s, layer, "gate_up"), 128), layer, "down")
    return x, hidden


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_decode_steps_equal_eager_ones(fp8: bool, device: torch.device) -> None:
    """A padded batch (five sequences, two rows of padding): a graph of the step, replayed with advancing positions,
    slots and lengths, against eager steps on a copy of the caches, all outputs and caches bit for bit."""
    page, m = 16, 7
    start = [300, 1, 17, 64, 1000]
    table, pages = kc.tables([n + 8 for n in start] + [0, 0], page)
    table[5:] = -1
    layers = _layers(2, device)
    host = [kc.cache(pages, KV_HEADS, page, D, torch.bfloat16, fp8, seed=i) for i in range(2)]
    mine, other = ([c.to(device) for c in host] for _ in range(2))
    angles = _table(D, 2048, device)
    x = torch.randn((m, H), generator=kc.gen("x")).bfloat16().to(device)
    positions, slots = torch.zeros(m, dtype=torch.int64, device=device), torch.zeros(m, dtype=torch.int64, device=device)
    lens, t = torch.zeros(m, dtype=torch.int32, device=device), table.to(device)

    def advance(step: int) -> None:
        at = torch.tensor([n + step for n in start])
        here = torch.cat([table[torch.arange(5), at // page].long() * page + at % page, torch.tensor([-1, -1])])
        positions.copy_(torch.cat([at, torch.tensor([0, 0])]))
        slots.copy_(here)
        lens.copy_(torch.cat([at + 1, torch.tensor([0, 0])]))

    advance(0)
    warm = [c.to(device) for c in host]
    _step(x, layers, warm, angles, positions, slots, t, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(x, layers, mine, angles, positions, slots, t, lens)
    for step in range(5):
        advance(step)
        graph.replay()
        want = _step(x, layers, other, angles, positions, slots, t, lens)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b) and torch.isfinite(a).all()
        for a, b in zip(mine, other):
            for u, w in zip(a, b):
                assert u is None or torch.equal(u.view(torch.uint8), w.view(torch.uint8))
        x.add_(0.125)
