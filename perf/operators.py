"""The FP8 operators with a scale for each block of 128, as cases to be timed, with their plain forms.

* ``linear``: ``fp8_block_linear``, e4m3 activations (a scale per row and 128 of K) times e4m3 weights
  (a scale per 128 x 128 block), 16-bit output;
* ``norm``: ``add_rmsnorm_fp8_quant``, the residual's addition, RMSNorm and e4m3 codes with scales;
* ``silu``: ``silu_mul_fp8_quant``, SiLU(gate) * up and e4m3 codes with scales;
* ``quant``: ``fp8_quant``, e4m3 codes with scales of a 16-bit activation.

``m`` counts rows (tokens); ``k`` is the length of a row that is multiplied, normalized or quantized,
``n`` the columns of a linear; ``group`` is 128, or 0 for one scale per row. Where ``own`` is true,
``run`` calls the operators of this package, else it computes them with elementary torch operations in
32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BLOCK = 128
E4M3_MAX = 448.0
MIN_SCALE = 1.0 / (448.0 * 512.0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# (n, k) of the four linears of the two decoders that the numerics suite and the benchmark use.
QWEN25_7B = {"qkv": (4608, 3584), "o": (3584, 3584), "gate_up": (37888, 3584), "down": (3584, 18944)}
QWEN25_05B = {"qkv": (1152, 896), "o": (896, 896), "gate_up": (9728, 896), "down": (896, 4864)}


def _linear(name, m, nk, dtype="fp16", bias=False, residual=False):
    return {"name": name, "kind": "linear", "m": m, "n": nk[0], "k": nk[1], "dtype": dtype, "bias": bias,
            "residual": residual}


def _rows(name, kind, m, k, dtype="fp16", group=BLOCK, residual=False):
    return {"name": name, "kind": kind, "m": m, "k": k, "dtype": dtype, "group": group, "residual": residual}


def listed():
    return [
        # Single-sequence decode: attention's output on its way to the o projection. Latency alone.
        _rows("quant_m1", "quant", 1, 3584),
        # A long prompt's attention output, an odd number of rows.
        _rows("quant_m4095", "quant", 4095, 3584, "bf16"),
        # Single-sequence decode: the residual's addition and the norm before gate_up.
        _rows("norm_m1", "norm", 1, 3584, residual=True),
        # A long prompt, the same step.
        _rows("norm_m4095", "norm", 4095, 3584, "bf16", residual=True),
        # A small decoder's MLP activation for three sequences, one scale per row (what w4a8_linear reads).
        _rows("silu_row_m3", "silu", 3, 4864, group=0),
        # The MLP activation of a long prompt.
        _rows("silu_m2048", "silu", 2048, 18944, "bf16"),
        # Single-sequence decode: the QKV projection with its bias.
        _linear("decode_qkv_m1", 1, QWEN25_7B["qkv"], bias=True),
        # A handful of sequences, the longest reduction, with the residual's addition.
        _linear("batch_down_m7", 7, QWEN25_7B["down"], "bf16", residual=True),
        # A serving batch of some dozens of sequences, the widest layer.
        _linear("batch_gate_up_m48", 48, QWEN25_7B["gate_up"]),
        # A short prompt through a layer whose sizes no block divides.
        _linear("ragged_m333", 333, (1000, 1296), "bf16", bias=True),
        # A prompt of ordinary length, the longest reduction.
        _linear("prefill_down_m1000", 1000, QWEN25_7B["down"], residual=True),
        # A long prompt: the largest product.
        _linear("prefill_gate_up_m4096", 4096, QWEN25_7B["gate_up"], "bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choices(("linear", "norm", "silu", "quant"), (8, 3, 3, 2))[0]
    dtype = rng.choice(("fp16", "bf16"))
    if kind != "linear":
        # Mostly whole blocks, now and then a row length that neither a block nor a load divides.
        k = _log_int(rng, 128, 8192 if kind == "norm" else 18944, rng.choice((128, 128, 128, 8, 1)))
        m = min(_log_int(rng, 1, 8192), 2048 * 18944 // k)
        c = _rows("", kind, m, k, dtype, rng.choice((128, 128, 0)), kind == "norm" and rng.random() < 0.8)
    else:
        decoder = rng.choice((QWEN25_7B, QWEN25_05B, None))
        if decoder is not None:
            n, k = decoder[rng.choice(("qkv", "o", "gate_up", "down"))]
        else:  # a layer of some other decoder, now and then with sizes that no block divides
            n = _log_int(rng, 64, 32768, rng.choice((128, 128, 16, 1)))
            k = _log_int(rng, 256, 16384, rng.choice((128, 128, 16)))
        m = min(_log_int(rng, 1, 4096), 4096 * 37888 * 3584 // (n * k))
        c = _linear("", m, (n, k), dtype, rng.random() < 0.3, rng.random() < 0.4)
    del c["name"]
    return c


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    m, k = case["m"], case["k"]
    if case["kind"] == "linear":
        n = case["n"]
        moved = m * k + n * k + 4 * (m + _blocks(n)) * _blocks(k) + 2 * m * n * (2 if case["residual"] else 1)
        return {"bytes": moved + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    scales = 4 * m * (_blocks(k) if case["group"] else 1)
    read = {"quant": 2 * m * k, "silu": 4 * m * k, "norm": (4 if case["residual"] else 2) * m * k + 2 * k}
    hidden = 2 * m * k if case["residual"] else 0
    return {"bytes": read[case["kind"]] + m * k + hidden + scales,
            "flops": m * k * {"quant": 3, "silu": 8, "norm": 7}[case["kind"]]}


# ----------------------------------------------------------------------------- inputs


def _activation(m, k, dtype, gen, scale=1.0):
    """Roughly normal values, a few channels twenty times larger, as a decoder's hidden states have."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    x[:, :: max(1, k // 8)] *= 20.0
    return (x * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, dtype = case["m"], case["k"], DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype}
    if case["kind"] == "linear":
        n = case["n"]
        state["x8"], state["x_scale"] = _plain_quant(_activation(m, k, torch.float32, gen), BLOCK)
        # The codes of a normal weight, scaled so that a block's largest is near the format's, and the
        # scales that give it a standard deviation of about 0.02.
        w = torch.randn((n, k), generator=gen, device="cuda", dtype=torch.float16).mul_(106.0)
        state["weight"] = w.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        state["w_scale"] = (torch.rand((_blocks(n), _blocks(k)), generator=gen, device="cuda") + 0.5) * 2e-4
        state["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype) if case["bias"] else None
        state["residual"] = torch.randn((m, n), generator=gen, device="cuda").to(dtype) if case["residual"] else None
    elif case["kind"] == "silu":
        state["x"] = _activation(m, 2 * k, dtype, gen)
    else:
        state["x"] = _activation(m, k, dtype, gen)
        if case["kind"] == "norm":
            state["residual"] = _activation(m, k, dtype, gen, 4.0) if case["residual"] else None
            state["weight"] = (1.0 + 0.1 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
    return state


# ----------------------------------------------------------------------------- plain forms


def _plain_quant(y, group):
    """Codes and scales of fp32 ``y [m, k]``: scale = max(amax / 448, 1 / (448 * 512)) over each 128 of a
    row (the last one shorter where 128 does not divide k), or over the row."""
    m, k = y.shape
    g = group or k
    nb = -(-k // g)
    padded = torch.nn.functional.pad(y, (0, nb * g - k)).reshape(m, nb, g)
    s = (padded.abs().amax(-1) / E4M3_MAX).clamp(min=MIN_SCALE)
    q = (padded / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(m, nb * g)[:, :k]
    return q.to(torch.float8_e4m3fn), s


def _spread(s, rows, cols):
    """Block scales ``[ceil(rows / 128), ceil(cols / 128)]`` as one value per element."""
    return s.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _plain(state):
    case, dtype = state["case"], state["dtype"]
    m, k = case["m"], case["k"]
    if case["kind"] == "linear":
        n = case["n"]
        x = state["x8"].float() * state["x_scale"].repeat_interleave(BLOCK, 1)[:, :k]
        y = x @ (state["weight"].float() * _spread(state["w_scale"], n, k)).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(dtype)
    x = state["x"].float()
    if case["kind"] == "quant":
        return _plain_quant(x, case["group"])
    if case["kind"] == "silu":
        gate, up = x[:, :k], x[:, k:]
        return _plain_quant(gate / (1.0 + torch.exp(-gate)) * up, case["group"])
    # The norm reads the hidden state as it is stored for the next residual, in 16 bits.
    hidden = state["x"] if state["residual"] is None else (x + state["residual"].float()).to(dtype)
    h = hidden.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * state["weight"].float()
    out = _plain_quant(y, case["group"])
    return out if state["residual"] is None else (*out, hidden)


def _own(state):
    case = state["case"]
    ops = torch.ops.tokenforge
    if case["kind"] == "linear":
        return ops.fp8_block_linear(state["x8"], state["x_scale"], state["weight"], state["w_scale"], state["bias"],
                                    state["dtype"], "hip", "none" if state["residual"] is None else "residual",
                                    state["residual"])
    if case["kind"] == "quant":
        return ops.fp8_quant(state["x"], case["group"])
    if case["kind"] == "silu":
        return ops.silu_mul_fp8_quant(state["x"], case["group"])
    q, s, hidden = ops.add_rmsnorm_fp8_quant(state["x"], state["residual"], state["weight"], EPS, case["group"])
    return (q, s) if state["residual"] is None else (q, s, hidden)


def run(state):
    if own:
        import tokenforge.kernels.ops  # noqa: F401  (registers torch.ops.tokenforge)

        return _own(state)
    return _plain(state)


# ----------------------------------------------------------------------------- 64 bits


def _exact_quant(y, group):
    """Codes (as values) and scales from the definition: a value v = y / s between 2^e and 2^(e + 1) goes
    to the nearest multiple of 2^(e - 3), ties to even, with e = -6 below 2^-6."""
    qs, ss = [], []
    for part in y.split(group or y.shape[1], dim=1):
        s = part.abs().max(dim=1, keepdim=True).values / E4M3_MAX
        s = torch.where(s < MIN_SCALE, torch.full_like(s, MIN_SCALE), s)
        v = part / s
        e = torch.frexp(v.abs()).exponent.sub(1).clamp(min=-6)
        step = torch.ldexp(torch.ones_like(v), e - 3)
        qs.append((torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX))
        ss.append(s)
    return torch.cat(qs, 1), torch.cat(ss, 1)


def exact(case, seed):
    state = prepare(case, seed)
    m, k = case["m"], case["k"]
    if case["kind"] == "linear":
        n = case["n"]
        rows = torch.arange(n, device="cuda") // BLOCK
        y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
        for b in range(_blocks(k)):
            at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            part = state["x8"][:, at].double() @ state["weight"][:, at].double().t()
            y += part * state["x_scale"][:, b, None].double() * state["w_scale"][rows, b].double()
        for extra in (state["bias"], state["residual"]):
            y = y if extra is None else y + extra.double()
        return y
    x = state["x"].double()
    if case["kind"] == "quant":
        return _exact_quant(x, case["group"])
    if case["kind"] == "silu":
        return _exact_quant(x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:], case["group"])
    h = x
    if state["residual"] is not None:
        h = (x + state["residual"].double()).to(state["dtype"]).double()
    mean = (h * h).sum(1, keepdim=True) / k
    out = _exact_quant(h / (mean + EPS).sqrt() * state["weight"].double(), case["group"])
    return out if state["residual"] is None else (*out, x + state["residual"].double())
