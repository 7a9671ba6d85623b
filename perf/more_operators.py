"""The key-value cache and the attention that reads it, as cases to be timed, with their plain forms.

* ``write``: ``kv_cache_write``, new tokens' keys and values into the slots of a paged cache, as 16-bit
  values or as e4m3 codes with a scale per token and head;
* ``rope``: ``rope_kv_cache_write``, the same with queries and keys rotated by their positions first;
* ``read``: ``kv_cache_read``, cached tokens by their slots, in 16 bits;
* ``attn``: ``paged_attention``, one new token of each sequence over its cached tokens.

``m`` counts tokens (``attn``: sequences), ``hq`` and ``hkv`` are query and key-value heads of length ``d``,
``page`` the tokens of a page; ``fp8`` says whether the cache holds e4m3 codes, ``tokens_first`` whether a
page's memory goes by token and then head rather than by head and then token. Where ``own`` is true, ``run``
calls the operators of this package, else it computes them with elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 1.0 / (448.0 * 512.0)
ROPE_BASE = 1e6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# (query heads, key-value heads, head length) of the two decoders that the numerics suite uses.
QWEN25_7B = (28, 4, 128)
QWEN25_05B = (14, 2, 64)


def _attn(name, m, heads, dtype, fp8, page, shortest, longest, window=0, tokens_first=False):
    return {"name": name, "kind": "attn", "m": m, "hq": heads[0], "hkv": heads[1], "d": heads[2], "dtype": dtype,
            "fp8": fp8, "page": page, "shortest": shortest, "longest": longest, "window": window,
            "tokens_first": tokens_first}


def _rows(name, kind, m, heads, dtype, fp8, page, rot=0, interleaved=False, tokens_first=False):
    return {"name": name, "kind": kind, "m": m, "hq": heads[0], "hkv": heads[1], "d": heads[2], "dtype": dtype,
            "fp8": fp8, "page": page, "rot": rot, "interleaved": interleaved, "tokens_first": tokens_first}


def listed():
    return [
        # A small decoder at the start of a single conversation: latency alone.
        _attn("attn_one_short", 1, QWEN25_05B, "fp16", False, 16, 33, 33),
        # A single conversation far into a long document: few heads, a long cache in 8 bits.
        _attn("attn_one_long", 1, QWEN25_7B, "bf16", True, 16, 32749, 32749),
        # A serving batch of unlike lengths over a 16-bit cache.
        _attn("attn_batch", 32, QWEN25_7B, "bf16", False, 16, 60, 4096),
        # A large batch over a cache in 8 bits with larger pages.
        _attn("attn_batch_fp8", 128, QWEN25_7B, "bf16", True, 64, 100, 2048),
        # A head of its own for each query, an odd head length, pages no tile divides, a window.
        _attn("attn_window_odd", 7, (12, 12, 80), "fp16", False, 24, 1, 5000, window=1023, tokens_first=True),
        # The largest: long documents, many at once.
        _attn("attn_long_batch", 64, QWEN25_7B, "bf16", False, 16, 2000, 16384),
        # A decode batch's new tokens into a 16-bit cache, without rotation.
        _rows("write_m64", "write", 64, QWEN25_05B, "fp16", False, 16),
        # A prompt's tokens into a cache in 8 bits.
        _rows("write_m4095_fp8", "write", 4095, QWEN25_7B, "bf16", True, 16),
        # Single-sequence decode: the rotation and the write in 8 bits. Latency alone.
        _rows("rope_m1_fp8", "rope", 1, QWEN25_7B, "bf16", True, 16, rot=128),
        # A long prompt into a 16-bit cache.
        _rows("rope_m8191", "rope", 8191, QWEN25_7B, "bf16", False, 64, rot=128),
        # A short prefix read back for the next part of a prompt.
        _rows("read_m333_fp8", "read", 333, QWEN25_05B, "fp16", True, 16),
        # A long prefix read back.
        _rows("read_m32767_fp8", "read", 32767, QWEN25_7B, "bf16", True, 16),
    ]


PADDED = 64 * 16384  # sequences times the longest length of the largest case


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("attn", "write", "rope", "read"), (6, 2, 3, 2))[0]
    heads = rng.choice((QWEN25_7B, QWEN25_7B, QWEN25_05B, None))
    if heads is None:  # some other decoder: one query a group up to one key-value head for all
        hkv = rng.choice((1, 2, 4, 8, 12))
        heads = (hkv * rng.choice((1, 2, 4, 5, 8, 20)), hkv, rng.choice((64, 80, 96, 128, 192, 256)))
    dtype, fp8 = rng.choice(("fp16", "bf16")), rng.random() < 0.5
    page, tokens_first = rng.choice((16, 16, 32, 64, 128, 8, 24)), rng.random() < 0.3
    if kind == "attn":
        m, longest = _log_int(rng, 1, 256), _log_int(rng, 16, 65536)
        spread, window = rng.choice((0.02, 0.3, 1)), rng.choice((0, 0, 0, 0.3))
        most = work(next(c for c in listed() if c["name"] == "attn_long_batch"))
        while True:  # shorter and fewer until it costs no more than the largest, padded or not
            c = _attn("", m, heads, dtype, fp8, page, max(1, int(longest * spread)), longest,
                      window and max(1, int(longest * window)), tokens_first)
            padded = m * longest * heads[1] * heads[2] <= PADDED * 4 * 128 and m * longest * heads[0] <= PADDED * 28
            if padded and all(work(c)[k] <= most[k] for k in most):
                break
            m, longest = max(1, m * 3 // 4), max(1, longest * 3 // 4)
        del c["name"]
        return c
    m = _log_int(rng, 1, 32767 if kind == "read" else 8191)
    m = min(m, 32767 * 28 * 128 // (4 * heads[0] * heads[2]))
    rot = rng.choice((heads[2], heads[2], heads[2] // 2)) if kind == "rope" else 0
    c = _rows("", kind, m, heads, dtype, fp8, page, rot, kind == "rope" and rng.random() < 0.3, tokens_first)
    del c["name"]
    return c


def _lens(case):
    """A length for each sequence between the case's shortest and longest, spread over the logarithm in an order
    of no pattern (steps of the golden ratio); the first is the longest."""
    a, b = math.log(case["shortest"]), math.log(case["longest"])
    at = [(1.0 + 0.6180339887498949 * i) % 1.0 for i in range(case["m"])]
    return [case["longest"] if i == 0 else max(1, int(math.exp(a + (b - a) * f))) for i, f in enumerate(at)]


def _cached_bytes(case):
    """Bytes of one cached token: keys and values, with their scales."""
    return 2 * case["hkv"] * (case["d"] + 4 if case["fp8"] else 2 * case["d"])


def work(case):
    m, hq, hkv, d = case["m"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "attn":
        lens = [min(n, case["window"]) if case["window"] else n for n in _lens(case)]
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": sum(lens) * _cached_bytes(case) + 4 * m * hq * d + 4 * pages + 4 * m,
                "flops": sum(lens) * hq * (4 * d + 5)}
    moved = m * (_cached_bytes(case) + 4 * hkv * d + 8)
    if case["kind"] == "rope":
        return {"bytes": moved + m * (4 * hq * d + 4 * case["rot"] + 8),
                "flops": m * (3 * (hq + hkv) * case["rot"] + (6 * hkv * d if case["fp8"] else 0))}
    return {"bytes": moved, "flops": m * hkv * d * (6 if case["fp8"] else 2)}


# ----------------------------------------------------------------------------- inputs


def _normal(shape, gen, scale=1.0):
    """Roughly normal values, a few channels eight times larger, as a decoder's keys have."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x[..., :: max(1, shape[-1] // 4)] *= 8.0
    return x * scale


def _cache(pages, case, gen):
    """A cache that is in use: (k_cache, v_cache, k_scale, v_scale), the caches [pages, hkv, page, d]."""
    hkv, page, d, dtype = case["hkv"], case["page"], case["d"], DTYPES[case["dtype"]]
    out, scales = [], []
    for size in (0.5, 1.0):
        shape = (pages, page, hkv, d) if case["tokens_first"] else (pages, hkv, page, d)
        x = torch.empty(shape, dtype=torch.float8_e4m3fn if case["fp8"] else dtype, device="cuda")
        s = torch.empty(shape[:-1], device="cuda") if case["fp8"] else None
        for part in range(0, pages, 1 << 14):  # a part at a time, for the memory of the values in 32 bits
            at = slice(part, min(pages, part + (1 << 14)))
            y = _normal((at.stop - at.start, *shape[1:]), gen, size)
            if case["fp8"]:
                x[at], s[at] = _plain_quant(y)
            else:
                x[at] = y.to(dtype)
        if case["tokens_first"]:
            x, s = x.transpose(1, 2), None if s is None else s.transpose(1, 2)
        out.append(x)
        scales.append(s)
    return (*out, *scales)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    m, hq, hkv, d, page, dtype = (case[k] for k in ("m", "hq", "hkv", "d", "page", "dtype"))
    dtype = DTYPES[dtype]
    state = {"case": case, "dtype": dtype}
    if case["kind"] == "attn":
        lens = torch.tensor(_lens(case), dtype=torch.int64)
        need = -(-lens // page)
        total, width = int(need.sum()), int(need.max())
        pages = total + 3
        order = torch.randperm(pages, generator=gen, device="cuda")[:total].to(torch.int32)
        first = (need.cumsum(0) - need).to("cuda")
        at = first[:, None] + torch.arange(width, device="cuda")
        held = torch.arange(width, device="cuda") < need.to("cuda")[:, None]
        state["block_table"] = torch.where(held, order[at.clamp(max=total - 1)], -1)
        state["seq_lens"] = lens.to(torch.int32).to("cuda")
        # the query as the first columns of a joined projection
        state["q"] = _normal((m, (hq + 2 * hkv) * d), gen).to(dtype)[:, : hq * d].unflatten(1, (hq, d))
        state["scale"] = d**-0.5
    else:
        pages = (m + m // 4) // page + 2
        state["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[:m]
        if case["kind"] != "read":  # tokens in order within their pages, as a sequence is laid out
            state["slots"] = state["slots"].sort().values
            qkv = _normal((m, (hq + 2 * hkv) * d), gen).to(dtype)
            parts = qkv.split((hq * d, hkv * d, hkv * d), dim=1)
            state["q"], state["k"], state["v"] = (p.unflatten(1, (-1, d)) for p in parts)
        if case["kind"] == "rope":
            # angles in 64 bits: a far position times the highest frequency has no fraction left in 32
            rot, far = case["rot"], 131072
            freq = ROPE_BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
            angle = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * freq
            state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
            start = int(torch.randint(0, far - m, (1,), generator=gen, device="cuda"))
            state["positions"] = torch.arange(start, start + m, device="cuda")
    state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"] = _cache(pages, case, gen)
    return state


# ----------------------------------------------------------------------------- plain forms


def _plain_quant(y):
    """Codes and scales of fp32 ``y [..., d]``: scale = max(amax / 448, 1 / (448 * 512)) over the last axis."""
    s = (y.abs().amax(-1) / E4M3_MAX).clamp(min=MIN_SCALE)
    return (y / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def _plain_rotate(x, cos_sin, interleaved):
    """fp32 ``x [m, h, d]`` with its first elements turned, by the pairs' angles ``cos_sin [m, rot]``."""
    cos, sin = cos_sin[:, None].chunk(2, dim=-1)
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_write(values, cache, scale, slots):
    page = cache.shape[2]
    at, off = slots // page, slots % page
    if scale is None:
        cache[at, :, off] = values.to(cache.dtype)
        return
    codes, s = _plain_quant(values)
    cache.view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
    scale[at, :, off] = s


def _plain_read(cache, scale, at, off):
    """fp32 values of the tokens at pages ``at`` and offsets ``off``: [*at.shape, hkv, d]."""
    if scale is None:
        return cache[at, :, off].float()
    codes = cache.view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn)
    return codes.float() * scale[at, :, off][..., None]


def _plain_attention(state):
    q, table, lens, window = state["q"].float(), state["block_table"], state["seq_lens"], state["case"]["window"]
    m, hq, d = q.shape
    page, hkv = state["k_cache"].shape[2], state["k_cache"].shape[1]
    pos = torch.arange(table.shape[1] * page, device="cuda")
    at, off = table[:, pos // page].long().clamp(min=0), (pos % page).expand(m, -1)
    seen = pos < lens[:, None]
    if window:
        seen = seen & (pos >= lens[:, None] - window)
    k = _plain_read(state["k_cache"], state["k_scale"], at, off).permute(0, 2, 3, 1)
    s = (q.unflatten(1, (hkv, hq // hkv)) @ k) * state["scale"]
    del k
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    v = _plain_read(state["v_cache"], state["v_scale"], at, off).transpose(1, 2)
    return ((p @ v) / p.sum(-1, keepdim=True)).flatten(1, 2).to(state["dtype"])


def _written(state):
    out = (state["k_cache"], state["v_cache"])
    return out if state["k_scale"] is None else (*out, state["k_scale"], state["v_scale"])


def _plain(state):
    case, dtype = state["case"], state["dtype"]
    if case["kind"] == "attn":
        return _plain_attention(state)
    slots, page = state["slots"], case["page"]
    if case["kind"] == "read":
        return tuple(_plain_read(state[f"{n}_cache"], state[f"{n}_scale"], slots // page, slots % page).to(dtype)
                     for n in "kv")
    q, k, v = (state[n].float() for n in "qkv")
    if case["kind"] == "rope":
        turn = state["cos_sin"][state["positions"]]
        q, k = _plain_rotate(q, turn, case["interleaved"]), _plain_rotate(k, turn, case["interleaved"])
    _plain_write(k, state["k_cache"], state["k_scale"], slots)
    _plain_write(v, state["v_cache"], state["v_scale"], slots)
    return (q.to(dtype), *_written(state)) if case["kind"] == "rope" else _written(state)


def _own(state):
    case = state["case"]
    ops = torch.ops.tokenforge
    cache = (state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])
    if case["kind"] == "attn":
        return ops.paged_attention(state["q"], *cache, state["block_table"], state["seq_lens"], state["scale"],
                                   case["window"])
    if case["kind"] == "read":
        return ops.kv_cache_read(*cache, state["slots"], state["dtype"])
    if case["kind"] == "write":
        ops.kv_cache_write(state["k"], state["v"], *cache, state["slots"])
        return _written(state)
    q = ops.rope_kv_cache_write(state["q"], state["k"], state["v"], state["cos_sin"], state["positions"], *cache,
                                state["slots"], case["interleaved"])
    return (q, *_written(state))


def run(state):
    if own:
        import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)

        return _own(state)
    return _plain(state)


# ----------------------------------------------------------------------------- 64 bits


def _exact_codes(y):
    """Codes (as values) and scales from the definition: a value v = y / s between 2^e and 2^(e + 1) goes
    to the nearest multiple of 2^(e - 3), ties to even, with e = -6 below 2^-6."""
    s = y.abs().max(dim=-1).values / E4M3_MAX
    s = torch.where(s < MIN_SCALE, torch.full_like(s, MIN_SCALE), s)
    v = y / s[..., None]
    e = torch.frexp(v.abs()).exponent.sub(1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX), s


def _exact_turn(x, state):
    """Each pair as a complex number times e^(i angle)."""
    case, rot = state["case"], state["case"]["rot"]
    z = state["cos_sin"][state["positions"]].double()
    z = torch.complex(z[:, : rot // 2], z[:, rot // 2 :])[:, None]
    first = torch.arange(rot // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else rot // 2)
    w = torch.complex(x[..., first], x[..., second]) * z
    out = x.clone()
    out[..., first], out[..., second] = w.real, w.imag
    return out


def exact(case, seed):
    state = prepare(case, seed)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    values = {}
    for n in "kv":  # tokens in the order of their slots: [pages * page, hkv, d]
        x = state[f"{n}_cache"].transpose(1, 2).reshape(-1, hkv, d)
        values[n] = (x, None if state[f"{n}_scale"] is None else state[f"{n}_scale"].transpose(1, 2).reshape(-1, hkv))

    def taken(n, slots):
        x, s = values[n]
        if s is None:
            return x[slots].double()
        return x.view(torch.uint8)[slots].view(torch.float8_e4m3fn).double() * s[slots].double()[..., None]

    if case["kind"] == "attn":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(state["seq_lens"].tolist()):
            pos = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
            slots = state["block_table"][b, pos // page].long() * page + pos % page
            k, v = taken("k", slots), taken("v", slots)
            for h in range(hkv):
                heads = slice(h * (case["hq"] // hkv), (h + 1) * (case["hq"] // hkv))
                s = state["q"][b, heads].double() @ k[:, h].t().contiguous() * state["scale"]
                out[b, heads] = torch.softmax(s, -1) @ v[:, h].contiguous()
        return out
    if case["kind"] == "read":
        return tuple(taken(n, state["slots"]) for n in "kv")
    q, k, v = (state[n].double() for n in "qkv")
    if case["kind"] == "rope":
        q, k = _exact_turn(q, state), _exact_turn(k, state)
    caches, scales = [], []
    for n, y in (("k", k), ("v", v)):
        x, s = values[n]
        x = x.double()
        if s is None:
            x[state["slots"]] = y
        else:
            s = s.double()
            x[state["slots"]], s[state["slots"]] = _exact_codes(y)
            scales.append(s.unflatten(0, (-1, page)).transpose(1, 2))
        caches.append(x.unflatten(0, (-1, page)).transpose(1, 2))
    return (q, *caches, *scales) if case["kind"] == "rope" else (*caches, *scales)
