"""Inputs and bounds of the cache's and the attention's tests."""

from __future__ import annotations

import dataclasses
import zlib

import numpy as np
import torch

from oracle import kv_cache as okv

F8 = torch.float8_e4m3fn
U32 = 2.0**-24
MFMA = 2.0**-23  # a matrix instruction's additions may cut instead of rounding
EPS = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step at most: finfo.eps / 2


def gen(*key: object) -> torch.Generator:
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


@dataclasses.dataclass
class Cache:
    """A cache in host memory; ``to`` gives the operators' arguments on a device."""

    k: torch.Tensor
    v: torch.Tensor
    ks: torch.Tensor | None
    vs: torch.Tensor | None
    tokens_first: bool = False

    def to(self, device: torch.device | str) -> tuple[torch.Tensor | None, ...]:
        def move(t: torch.Tensor | None) -> torch.Tensor | None:
            if t is None:
                return None
            if not self.tokens_first:
                return t.clone().to(device)
            return t.transpose(1, 2).contiguous().to(device).transpose(1, 2)

        return tuple(move(t) for t in (self.k, self.v, self.ks, self.vs))


def cache(pages: int, heads: int, page: int, d: int, dtype: torch.dtype, fp8: bool, seed: int = 0,
          tokens_first: bool = False) -> Cache:
    """A cache in use: normal values, some channels eight times larger; e4m3 codes of them with their scales."""
    g = gen("cache", pages, heads, page, d, seed)
    out = []
    for size in (0.5, 1.0):
        x = torch.randn((pages, heads, page, d), generator=g) * size
        x[..., ::max(1, d // 4)] *= 8.0
        if fp8:
            s = (x.abs().amax(-1) / 448.0).clamp(min=1 / (448.0 * 512.0))
            out.append(((x / s[..., None]).clamp(-448, 448).to(F8), s))
        else:
            out.append((x.to(dtype), None))
    (k, ks), (v, vs) = out
    return Cache(k, v, ks, vs, tokens_first)


def values(x: torch.Tensor) -> np.ndarray:
    return x.detach().cpu().double().numpy()


def tables(lens: list[int], page: int, width: int | None = None, seed: int = 0, spare: int = 2) -> tuple[torch.Tensor, int]:
    """Block tables of sequences of these lengths over pages in no order, -1 behind a sequence's last; and the pages."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen("pages", pages, seed)).to(torch.int32)
    table = torch.full((len(lens), max(width or 0, *need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def check_attention(out: torch.Tensor, q: torch.Tensor, c: Cache, table: torch.Tensor, lens: list[int], scale: float,
                    window: int = 0) -> None:
    """The attention's output against 64 bits.

    A score is a sum of d exact products in fp32: d + 1 additions, each off by at most MFMA of the products'
    magnitudes' sum; its scale, e4m3 scale and log2(e) are 4 roundings of the score (|score| <= that sum), the
    subtraction of the maximum and the exponential's own error 4 more of magnitudes up to twice that. So a
    probability is off by a factor within 1 + e, e = (d + 16) MFMA spread (to first order, and 2^-22 for the
    exponential), numerator and denominator alike: 2 e of the sum of p |v|. The probabilities' two halves: within
    2^-16 of each (8 bits cut, the rest rounded at 8 bits), the e4m3 scale's product U32. Both sums of n terms: n + 64
    additions (joins among them) within MFMA each, and the division. Then half a step of the result."""
    d, dtype, page = q.shape[2], q.dtype, c.k.shape[2]
    got = values(out)
    assert np.isfinite(got).all()
    kc, vc = values(c.k.float()), values(c.v.float())
    ks, vs = (None if s is None else values(s) for s in (c.ks, c.vs))
    for b, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * page)
        begin = max(0, n - window) if window else 0
        row = table[b].numpy()
        k, v = okv.tokens(kc, ks, row, begin, n), okv.tokens(vc, vs, row, begin, n)
        want, size, spread = okv.attention(values(q[b]), k, v, scale)
        e = (d + 16) * MFMA * spread[:, None] + 2.0**-22
        bound = (2 * e + 2.0**-16 + 2 * (k.shape[0] + 64) * MFMA) * size
        # half a step of the value that is rounded (and fp16's subnormal step)
        bound += EPS[dtype] * (np.abs(want) + bound) + (2.0**-25 if dtype == torch.float16 else 0.0)
        over = np.abs(got[b] - want) - bound
        assert over.max() <= 0, f"sequence {b} of {n}: {over.max():.3e} over the bound at {np.unravel_index(over.argmax(), over.shape)}"
