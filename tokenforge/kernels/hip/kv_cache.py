"""The paged key-value cache and the attention that reads it, on gfx950.

No counterpart in the reference, which has no attention. A cache is two tensors ``[pages, heads, page_size,
head_dim]`` (any strides that keep rows apart, so a cache laid out by token and then head goes in as its
transposed view), fp16 or bf16, or e4m3 codes with fp32 scales ``[pages, heads, page_size]``: a scale per
token and head, by the rule of the FP8 quantizers. Token ``i`` of page ``p`` is in slot ``p * page_size +
i``; a sequence's pages, in order, are a row of a block table.
"""

from __future__ import annotations

import ctypes

import torch

from tokenforge.kernels import _lib
from tokenforge.kernels.hip._common import on_device, ptr, require_gpu, stream_of
from tokenforge.kernels.hip.fp8_block import DTYPES

E4M3 = torch.float8_e4m3fn
MAX_HEAD_DIM = _lib.KV_MAX_HEAD_DIM
MAX_TOKEN_STRIDE = 1 << 24

Cache = tuple[torch.Tensor, torch.Tensor, "torch.Tensor | None", "torch.Tensor | None"]


# ----------------------------------------------------------------------------- checks


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no two elements of ``t`` share memory (dimensions nested by their strides)."""
    extent = 0
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride <= extent:
            return False
        extent += stride * (size - 1)
    return True


def _runs(t: torch.Tensor) -> tuple[list[tuple[int, int]], int]:
    """``t`` as runs of bytes: its dimensions of two or more as (stride in bytes, size), the largest stride first, and the
    bytes of a run (a cache's row, a scale)."""
    e = t.element_size()
    dims = [(st * e, sz) for st, sz in zip(t.stride()[:3], t.shape) if sz > 1]
    return sorted(dims, reverse=True), e * (t.shape[3] if t.dim() == 4 else 1)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors of nested dimensions (:func:`_rows_apart`) share memory. A dimension of one stride in both is settled
    by the one or two differences of its indices that bring what lies within it together; from one on where the
    strides differ, ranges that meet count as overlap."""
    (da, ra), (db, rb) = _runs(a), _runs(b)

    def meet(far: int, i: int) -> bool:
        ea, eb = (r + sum(st * (sz - 1) for st, sz in d[i:]) for d, r in ((da, ra), (db, rb)))
        if far >= ea or far <= -eb:
            return False
        if i >= len(da) or i >= len(db) or da[i][0] != db[i][0]:
            return True
        s, na = da[i]
        nb = db[i][1]
        ia, ib = ea - s * (na - 1), eb - s * (nb - 1)
        first, last = (-ib - far) // s + 1, (ia - 1 - far) // s
        return any(meet(far + s * t, i + 1) for t in range(max(first, 1 - na), min(last, nb - 1) + 1))

    return meet(b.data_ptr() - a.data_ptr(), 0)


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor | None,
                v_scale: torch.Tensor | None, *, written: bool = False) -> tuple[int, int, int, int]:
    """Checks of a cache, on any device; returns ``(pages, heads, page_size, head_dim)``."""
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be [pages, heads, page_size, head_dim], got {tuple(k_cache.shape)}")
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"v_cache shape {tuple(v_cache.shape)} != {tuple(k_cache.shape)}")
    if k_cache.dtype not in DTYPES and k_cache.dtype != E4M3:
        raise TypeError(f"the cache must be fp16, bf16 or float8_e4m3fn, got {k_cache.dtype}")
    if v_cache.dtype != k_cache.dtype:
        raise TypeError(f"v_cache must be {k_cache.dtype} like k_cache, got {v_cache.dtype}")
    pages, heads, page_size, d = k_cache.shape
    if 0 in (pages, heads, page_size):
        raise ValueError(f"the cache has no slots: {tuple(k_cache.shape)}")
    if heads > 65535 or page_size > 1 << 24:
        raise ValueError(f"at most 65535 heads and pages of 2^24 tokens are supported, got {tuple(k_cache.shape)}")
    if d == 0 or d % 8 or d > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    fp8 = k_cache.dtype == E4M3
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check_rows(name, t, 8 if fp8 else 16, written)
    if (k_scale is not None) != fp8 or (v_scale is not None) != fp8:
        raise ValueError("k_scale and v_scale go with a float8_e4m3fn cache, and only with it")
    if fp8:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            assert t is not None
            if tuple(t.shape) != (pages, heads, page_size):
                raise ValueError(f"{name} shape {tuple(t.shape)} != {(pages, heads, page_size)}")
            if t.dtype != torch.float32:
                raise TypeError(f"{name} must be fp32, got {t.dtype}")
            if page_size > 1 and t.stride(2) >= MAX_TOKEN_STRIDE:
                raise ValueError(f"{name}: a page's tokens must lie less than {MAX_TOKEN_STRIDE} elements apart")
            if written and not _rows_apart(t):
                raise ValueError(f"{name} is written and must not hold an element twice")
        if written and k_scale.data_ptr() == v_scale.data_ptr():  # type: ignore[union-attr]
            raise ValueError("k_scale and v_scale are written and must not be one tensor")
    if written and k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("k_cache and v_cache are written and must not be one tensor")
    if written:
        held = [(n, t) for n, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale),
                                    ("v_scale", v_scale)) if t is not None]
        for j, (name, t) in enumerate(held):
            for other, u in held[:j]:
                if _overlap(u, t):
                    raise ValueError(f"{other} and {name} are written and must not overlap")
    return pages, heads, page_size, d


def _check_rows(name: str, t: torch.Tensor, align: int, written: bool) -> None:
    if t.stride(3) != 1 and t.shape[3] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if any(st % 8 for st, sz in zip(t.stride()[:3], t.shape) if sz > 1) or t.data_ptr() % align:
        raise ValueError(f"rows of {name} must start on {align} bytes")
    if t.shape[2] > 1 and t.stride(2) >= MAX_TOKEN_STRIDE:
        raise ValueError(f"{name}: a page's tokens must lie less than {MAX_TOKEN_STRIDE} elements apart")
    if written and not _rows_apart(t):
        raise ValueError(f"{name} is written and must not hold an element twice")


def _check_tokens(name: str, x: torch.Tensor, shape: tuple[int, ...], k_cache: torch.Tensor,
                  dtype: torch.dtype | None = None) -> None:
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} shape {tuple(x.shape)} != {shape}")
    want = dtype if dtype is not None else (k_cache.dtype if k_cache.dtype != E4M3 else None)
    if x.dtype not in DTYPES or (want is not None and x.dtype != want):
        raise TypeError(f"{name} must be {want if want is not None else 'fp16 or bf16'}, got {x.dtype}")


def _check_index(name: str, t: torch.Tensor, size: int, dtype: torch.dtype) -> None:
    if tuple(t.shape) != (size,):
        raise ValueError(f"{name} shape {tuple(t.shape)} != {(size,)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def check_write(k: torch.Tensor, v: torch.Tensor, cache: Cache, slots: torch.Tensor) -> int:
    """Every check of the write, on any device; returns the tokens."""
    _, heads, _, d = check_cache(*cache, written=True)
    if k.dim() != 3:
        raise ValueError(f"k must be [tokens, heads, head_dim], got {tuple(k.shape)}")
    _check_tokens("k", k, (k.shape[0], heads, d), cache[0])
    _check_tokens("v", v, (k.shape[0], heads, d), cache[0], k.dtype)
    _check_index("slots", slots, k.shape[0], torch.int64)
    return k.shape[0]


def check_rope(q: torch.Tensor, k: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor) -> int:
    """The rotation's own checks (after :func:`check_write`); returns the rotated length."""
    t, _, d = k.shape
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] > 65535:
        raise ValueError(f"q must be [tokens, q_heads, head_dim], got {tuple(q.shape)}")
    _check_tokens("q", q, (t, q.shape[1], d), k, k.dtype)
    if cos_sin.dim() != 2 or cos_sin.shape[0] == 0:
        raise ValueError(f"cos_sin must be [max_positions, rot], got {tuple(cos_sin.shape)}")
    if cos_sin.dtype != torch.float32:
        raise TypeError(f"cos_sin must be fp32, got {cos_sin.dtype}")
    rot = cos_sin.shape[1]
    if rot == 0 or rot % 2 or rot > d:
        raise ValueError(f"cos_sin's rows must be even, above 0 and at most head_dim {d}, got {rot}")
    _check_index("positions", positions, t, torch.int64)
    return rot


def check_read(cache: Cache, slots: torch.Tensor, out_dtype: torch.dtype) -> int:
    """Every check of the read, on any device; returns the tokens."""
    check_cache(*cache)
    if out_dtype not in DTYPES or (cache[0].dtype != E4M3 and out_dtype != cache[0].dtype):
        want = "float16 or bfloat16" if cache[0].dtype == E4M3 else f"{cache[0].dtype} like the cache"
        raise TypeError(f"out_dtype must be {want}, got {out_dtype}")
    _check_index("slots", slots, slots.shape[0] if slots.dim() else 0, torch.int64)
    return slots.shape[0]


def check_attention(q: torch.Tensor, cache: Cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    window: int) -> int:
    """Every check of the attention, on any device; returns the sequences."""
    _, heads, page_size, d = check_cache(*cache)
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % heads or q.shape[1] > 65535:
        raise ValueError(f"q must be [sequences, a multiple of {heads} heads, head_dim], got {tuple(q.shape)}")
    m = q.shape[0]
    _check_tokens("q", q, (m, q.shape[1], d), cache[0])
    if block_table.dim() != 2 or block_table.shape[0] != m:
        raise ValueError(f"block_table must be [{m}, pages], got {tuple(block_table.shape)}")
    if block_table.dtype != torch.int32:
        raise TypeError(f"block_table must be torch.int32, got {block_table.dtype}")
    _check_index("seq_lens", seq_lens, m, torch.int32)
    if window < 0:
        raise ValueError(f"window must be 0 (none) or more, got {window}")
    width = block_table.shape[1]
    group = q.shape[1] // heads
    items = m * heads * -(-group // (32 if group > 16 and d <= 128 else 16))  # query heads that share a pass, as the C entry
    if width > 0x7FFFFF00 // page_size or m * q.shape[1] > 0x7FFFFF or items * -(-width * page_size // 16) > 0x7FFFFFFF:
        raise ValueError(f"{m} sequences of {width} pages of {page_size} with {q.shape[1]} heads are too large")
    return m


# ----------------------------------------------------------------------------- launches


def _strides(t: torch.Tensor | None) -> ctypes.Array[ctypes.c_int64]:
    """Strides of (page, head, token); those of a dimension of one are never multiplied by anything but 0."""
    s = (0, 0, 0) if t is None else tuple(st if sz > 1 else 0 for st, sz in zip(t.stride()[:3], t.shape))
    return (ctypes.c_int64 * 3)(*s)


def to_c_cache(cache: Cache) -> _lib.TfKvCache:
    k, v, ks, vs = cache
    pages, heads, page_size, d = k.shape
    return _lib.TfKvCache(k.data_ptr(), v.data_ptr(), ptr(ks), ptr(vs), pages, heads, page_size, d,
                          _lib.DTYPE_E4M3 if k.dtype == E4M3 else DTYPES[k.dtype], _strides(k), _strides(v),
                          _strides(ks), _strides(vs))


def _head_rows(x: torch.Tensor) -> torch.Tensor:
    """``x [tokens, heads, head_dim]`` with rows contiguous and on 16 bytes; a copy only when needed."""
    ok = x.stride(2) == 1 and x.data_ptr() % 16 == 0
    if ok and all(st % 8 == 0 for st, sz in zip(x.stride()[:2], x.shape) if sz > 1):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _two(x: torch.Tensor) -> tuple[int, int]:
    return (x.stride(0) if x.shape[0] > 1 else 0, x.stride(1) if x.shape[1] > 1 else 0)


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, cache: Cache, slots: torch.Tensor) -> None:
    """Keys and values ``[T, heads, head_dim]`` into their slots (``tf_kv_cache_write``)."""
    t = check_write(k, v, cache, slots)
    dev = require_gpu("kv_cache_write", *(x for x in (k, v, *cache, slots) if x is not None))
    if t == 0:
        return
    k, v, slots = _head_rows(k), _head_rows(v), slots.contiguous()
    c = to_c_cache(cache)
    with on_device(dev):
        rc = _lib.lib().tf_kv_cache_write(ctypes.byref(c), k.data_ptr(), *_two(k), v.data_ptr(), *_two(v),
                                          DTYPES[k.dtype], slots.data_ptr(), t, stream_of(dev))
    _lib.check(rc, "tf_kv_cache_write")


def rope_kv_cache_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos_sin: torch.Tensor,
                        positions: torch.Tensor, cache: Cache, slots: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """:func:`kv_cache_write` with q and k rotated first; returns the rotated q (``tf_rope_kv_cache_write``)."""
    t = check_write(k, v, cache, slots)
    rot = check_rope(q, k, cos_sin, positions)
    dev = require_gpu("rope_kv_cache_write",
                      *(x for x in (q, k, v, cos_sin, positions, *cache, slots) if x is not None))
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if t == 0:
        return out
    q, k, v = _head_rows(q), _head_rows(k), _head_rows(v)
    slots, positions = slots.contiguous(), positions.contiguous()
    if not cos_sin.is_contiguous() or cos_sin.data_ptr() % 16:
        cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
    c = to_c_cache(cache)
    with on_device(dev):
        rc = _lib.lib().tf_rope_kv_cache_write(
            ctypes.byref(c), q.data_ptr(), *_two(q), q.shape[1], k.data_ptr(), *_two(k), v.data_ptr(), *_two(v),
            DTYPES[k.dtype], cos_sin.data_ptr(), cos_sin.shape[0], rot, int(interleaved), positions.data_ptr(),
            slots.data_ptr(), out.data_ptr(), t, stream_of(dev))
    _lib.check(rc, "tf_rope_kv_cache_write")
    return out


def kv_cache_read(cache: Cache, slots: torch.Tensor, out_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[T, heads, head_dim]`` of the tokens in ``slots`` (``tf_kv_cache_read``)."""
    t = check_read(cache, slots, out_dtype)
    dev = require_gpu("kv_cache_read", *(x for x in (*cache, slots) if x is not None))
    shape = (t, cache[0].shape[1], cache[0].shape[3])
    k, v = (torch.empty(shape, dtype=out_dtype, device=dev) for _ in range(2))
    if t:
        slots = slots.contiguous()
        c = to_c_cache(cache)
        with on_device(dev):
            rc = _lib.lib().tf_kv_cache_read(ctypes.byref(c), slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                                             DTYPES[out_dtype], t, stream_of(dev))
        _lib.check(rc, "tf_kv_cache_read")
    return k, v


def paged_attention(q: torch.Tensor, cache: Cache, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                    window: int) -> torch.Tensor:
    """One query token per sequence over its cached tokens (``tf_paged_attention``)."""
    m = check_attention(q, cache, block_table, seq_lens, window)
    dev = require_gpu("paged_attention", *(x for x in (q, *cache, block_table, seq_lens) if x is not None))
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if m == 0:
        return out
    q, seq_lens = _head_rows(q), seq_lens.contiguous()
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    c = to_c_cache(cache)
    width = block_table.shape[1]
    window = min(window, 0x7FFFFFFF)
    need = int(_lib.lib().tf_paged_attention_workspace_bytes(ctypes.byref(c), m, q.shape[1], width, window))
    ws = torch.empty((need + 3) // 4, dtype=torch.float32, device=dev) if need > 0 else None
    with on_device(dev):
        rc = _lib.lib().tf_paged_attention(
            ctypes.byref(c), q.data_ptr(), *_two(q), q.shape[1], DTYPES[q.dtype], block_table.data_ptr(),
            block_table.stride(0) if m > 1 else 0, width, seq_lens.data_ptr(), m, float(scale),
            window, out.data_ptr(), ptr(ws), need, stream_of(dev))
    _lib.check(rc, "tf_paged_attention")
    return out
