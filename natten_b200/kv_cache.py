"""The paged key/value cache and the serving form of causal 1-D neighborhood attention that reads it.

A cache is two pools of pages, ``[pages, page_size, heads_kv, head_dim]``; which page holds which tokens of
a sequence is the caller's table: token p of sequence b lies in page ``page_table[b, p // page_size]``, slot
``p % page_size``. Tables and lengths are int32 tensors on the GPU, read when the kernels run: nothing here
waits for the device, and a captured CUDA graph follows tables and lengths that change in place.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _native, ops
from .checks import _dim_arg
from .functional import _native_eligible, _require_cuda, _wants_grad

COMPUTE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
CACHE_DTYPES = COMPUTE_DTYPES + (torch.float8_e4m3fn,)
MAX_HEAD_DIM = 256


class KVCache(NamedTuple):
    """Pools of pages. With ``torch.float8_e4m3fn`` pools, ``key_scale`` and ``value_scale`` (fp32,
    ``[pages, page_size, heads_kv]``) hold one scale for each token and head; otherwise they are None.
    Scales are what `kv_cache_write` leaves there, 2**-126 or more, or NaN: attention works with a value
    scale's logarithm.

    Any strides with contiguous channels will do (a ``[pages, heads, page_size, head_dim]`` pool is passed
    as its transpose). Slots that no token was written to are never read."""
    key: Tensor
    value: Tensor
    key_scale: Optional[Tensor] = None
    value_scale: Optional[Tensor] = None

    @classmethod
    def allocate(cls, pages: int, page_size: int, heads_kv: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "KVCache":
        """An empty cache."""
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"A cache holds fp32, fp16, bf16 or e4m3, got {dtype}.")
        pools = [torch.empty(pages, page_size, heads_kv, head_dim, dtype=dtype, device=device)
                 for _ in range(2)]
        if dtype == torch.float8_e4m3fn:
            pools += [torch.empty(pages, page_size, heads_kv, dtype=torch.float32, device=device)
                      for _ in range(2)]
        return cls(*pools)


def _check_sizes(name: str, t: Tensor) -> None:
    if max(t.shape) >= 2 ** 31:
        raise NotImplementedError(f"`{name}` must have less than 2**31 entries along every axis, got "
                                  f"{tuple(t.shape)}.")


def _expect_cache(cache: KVCache) -> None:
    if not isinstance(cache, KVCache):
        raise ValueError(f"Expected a KVCache, got {type(cache)}.")


def _check_cache(cache: KVCache) -> None:
    key, value, *scales = cache
    if not isinstance(key, Tensor) or not isinstance(value, Tensor) or key.dim() != 4 or value.shape != key.shape:
        raise ValueError("A cache's pools are [pages, page_size, heads_kv, head_dim], keys and values "
                         "alike.")
    if key.dtype != value.dtype or key.device != value.device:
        raise ValueError("A cache's pools must have the same device and data type, got "
                         f"{key.device}, {value.device}, {key.dtype}, {value.dtype}.")
    if key.dtype not in CACHE_DTYPES:
        raise ValueError(f"A cache holds fp32, fp16, bf16 or e4m3, got {key.dtype}.")
    if min(key.shape[1:]) < 1:
        raise ValueError(f"A cache's pages, heads and channels cannot be empty, got {tuple(key.shape)}.")
    _check_sizes("cache", key)
    if key.shape[-1] > MAX_HEAD_DIM:
        raise NotImplementedError(f"The cache takes head dims up to {MAX_HEAD_DIM}, got {key.shape[-1]}.")
    if key.shape[-1] > 1 and (key.stride(-1) != 1 or value.stride(-1) != 1):
        raise ValueError("The channels of a cache's heads must be contiguous.")
    if key.dtype == torch.float8_e4m3fn:
        for s in scales:
            if s is None or s.shape != key.shape[:3] or s.dtype != torch.float32 or s.device != key.device:
                raise ValueError("An 8-bit cache needs fp32 scales [pages, page_size, heads_kv] on its "
                                 "device, for keys and for values.")
    elif scales[0] is not None or scales[1] is not None:
        raise ValueError(f"Only an 8-bit cache has scales, got {key.dtype}.")


def _check_rows(cache: KVCache, **tensors: Tensor) -> None:
    """Queries, keys and values: [B, T, heads, head_dim] in a type that the cache is read or written in."""
    for name, t in tensors.items():
        if t.dim() != 4 or t.shape[-1] != cache.key.shape[-1]:
            raise ValueError(f"`{name}` must be [batch, tokens, heads, {cache.key.shape[-1]}], got "
                             f"{tuple(t.shape)}.")
        _check_sizes(name, t)
        if t.device != cache.key.device:
            raise ValueError(f"`{name}` must be on the cache's device, got {t.device}.")
        _check_dtype(cache, t.dtype, name)


def _check_dtype(cache: KVCache, dtype: torch.dtype, name: str) -> None:
    if dtype not in COMPUTE_DTYPES or (cache.key.dtype in COMPUTE_DTYPES and dtype != cache.key.dtype):
        raise ValueError(f"`{name}` must have the cache's data type (fp32, fp16 or bf16 for an 8-bit "
                         f"cache), got {dtype} and {cache.key.dtype}.")


def _table(cache: KVCache, page_table: Tensor, batch: Optional[int]) -> Tensor:
    if (page_table.dim() != 2 or page_table.dtype != torch.int32
            or page_table.device != cache.key.device
            or (batch is not None and page_table.shape[0] != batch)):
        raise ValueError("`page_table` must be an int32 tensor [batch, pages of a sequence] on the cache's "
                         f"device, got {page_table.dtype} {tuple(page_table.shape)} on "
                         f"{page_table.device}.")
    _check_sizes("page_table", page_table)
    return page_table if page_table.stride(1) == 1 or page_table.shape[1] <= 1 else page_table.contiguous()


def _per_sequence(cache: KVCache, t: Optional[Tensor], batch: int, name: str) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != batch or t.dtype != torch.int32 or t.device != cache.key.device:
        raise ValueError(f"`{name}` must be an int32 tensor [{batch}] on the cache's device, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}.")
    return t.contiguous()


def _refuse_grad(what: str, *tensors: Tensor) -> None:
    if _wants_grad(*tensors):
        raise NotImplementedError(f"{what} is not differentiable: call it under torch.no_grad() or "
                                  "torch.inference_mode().")


def kv_cache_write(cache: KVCache, key: Tensor, value: Tensor, page_table: Tensor,
                   start: Optional[Tensor] = None, counts: Optional[Tensor] = None) -> None:
    """Writes ``[batch, tokens, heads_kv, head_dim]`` keys and values into the cache.

    Token t of sequence b goes to position ``start[b] + t`` (``t`` without ``start``), if ``t <
    counts[b]`` (all without ``counts``): what lies behind a padded sequence's tokens stays as it was. An
    8-bit cache quantises as it is written: ``scale = max(max|x| / 448, 2**-126)`` for each token and head,
    ``x / scale`` (both 32-bit divisions) rounded to the nearest e4m3; a row that holds a NaN or an infinity reads back as NaN.

    Positions that are negative, behind the table, or on a table entry outside ``[0, pages)`` are dropped.
    The slots of one call must be different ones: of two tokens on the same slot, which one (or a mixture)
    is left is undefined."""
    _expect_cache(cache)
    if (_native_eligible()
            and _native.kv_cache_write(cache, key, value, page_table, start, counts) is not None):
        return
    _check_cache(cache)
    _check_rows(cache, key=key, value=value)
    if key.shape != value.shape or key.shape[2] != cache.key.shape[2] or key.dtype != value.dtype:
        raise ValueError("Keys and values must be alike and have the cache's number of heads, got "
                         f"{tuple(key.shape)} {key.dtype}, {tuple(value.shape)} {value.dtype} and "
                         f"{cache.key.shape[2]} heads.")
    _refuse_grad("kv_cache_write()", key, value, *cache)
    if any(n > 1 and s == 0 for t in cache if t is not None for n, s in zip(t.shape, t.stride())):
        raise ValueError("kv_cache_write() needs pools with an element of their own in every place.")
    batch = key.shape[0]
    table = _table(cache, page_table, batch)
    start, counts = (_per_sequence(cache, t, batch, n) for t, n in ((start, "start"), (counts, "counts")))
    _require_cuda(*cache)
    ops.kv_cache_write(key, value, *cache, table, start, counts)


def kv_cache_read(cache: KVCache, page_table: Tensor, length: int, start: Optional[Tensor] = None,
                  counts: Optional[Tensor] = None,
                  dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """Reads tokens back: contiguous ``[batch, length, heads_kv, head_dim]`` keys and values, e.g. a cached
    prefix that a new chunk attends with `attention`. That takes no lengths, and a key of zeros has a weight
    like any other: read prefixes of equal length together, others one by one.

    Row t of sequence b is the token at ``start[b] + t`` (``t`` without ``start``); rows ``t >= counts[b]``
    and tokens that are on no page are zeros. ``dtype`` is the cache's, or fp32, fp16 or bf16 for an 8-bit
    cache (default bf16)."""
    _expect_cache(cache)
    if dtype is None:
        dtype = getattr(cache.key, "dtype", None)
        dtype = torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype
    if _native_eligible():
        result = _native.kv_cache_read(cache, page_table, length, start, counts, dtype)
        if result is not None:
            return result
    _check_cache(cache)
    _check_dtype(cache, dtype, "dtype")
    if not isinstance(length, int) or isinstance(length, bool) or not 0 <= length < 2 ** 31:
        raise ValueError(f"`length` must be a number of tokens, got {length!r}.")
    _refuse_grad("kv_cache_read()", *cache)
    table = _table(cache, page_table, None)
    start, counts = (_per_sequence(cache, t, table.shape[0], n)
                     for t, n in ((start, "start"), (counts, "counts")))
    _require_cuda(*cache)
    return ops.kv_cache_read(*cache, table, start, counts, length, dtype)


def na1d_decode(query: Tensor, cache: KVCache, page_table: Tensor, lengths: Tensor,
                kernel_size: Optional[int] = None, dilation: int = 1, scale: Optional[float] = None,
                return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Causal 1-D neighborhood attention of the newest tokens over a paged cache: what
    ``na1d(..., is_causal=True)`` (stride 1) gives for the last rows of each sequence, without the others.

    ``query`` is ``[batch, tokens, heads, head_dim]``, the newest tokens of every sequence (one in a
    decoding step, a few when drafted tokens are checked); ``lengths`` (int32, ``[batch]``) counts the
    tokens in the cache, the newest included: write them first. Query t stands at ``p = lengths - tokens +
    t`` and attends ``p, p - dilation, ...``: ``kernel_size`` tokens at most, as many as there are; all of
    them without ``kernel_size``. heads may be a multiple of the cache's. A query that attends no token
    (``p < 0`` for a sequence shorter than the number of queries, or no page) gives zeros and a logsumexp
    of -inf; tokens on table entries outside ``[0, pages)`` are left out, so pages behind a window can be
    given back.

    The cache has the query's data type or is an 8-bit one. Returns the output in the query's type, with
    ``return_lse`` also the logsumexp (fp32 ``[batch, tokens, heads]``), as `merge_attentions` takes them."""
    _expect_cache(cache)
    if _native_eligible():
        result = _native.na1d_decode(query, cache, page_table, lengths, kernel_size, dilation, scale,
                                     bool(return_lse))
        if result is not None:
            return result
    _check_cache(cache)
    _check_rows(cache, query=query)
    heads, heads_kv = query.shape[2], cache.key.shape[2]
    if heads < heads_kv or heads % heads_kv != 0:
        raise ValueError("Key/value heads must evenly divide query heads, got "
                         f"{heads=}, {heads_kv=}.")
    if kernel_size is not None:
        kernel_size, = _dim_arg(1, kernel_size, "kernel_size", 2, None)
    dilation, = _dim_arg(1, dilation, "dilation", 1, 1)
    scale = scale or query.shape[-1] ** -0.5
    if not 0 < scale < float("inf"):
        raise ValueError(f"`scale` must be a positive number, got {scale}.")
    _refuse_grad("na1d_decode()", query, *cache)
    table = _table(cache, page_table, query.shape[0])
    lengths = _per_sequence(cache, lengths, query.shape[0], "lengths")
    if lengths is None:
        raise ValueError("`lengths` must be an int32 tensor on the cache's device, got None.")
    _require_cuda(*cache)
    kernel_size, dilation = (min(n, 2 ** 31 - 1) for n in (kernel_size or 0, dilation))   # C ints
    out, lse = ops.na1d_decode(query, *cache, table, lengths, kernel_size, dilation, float(scale))
    return (out, lse) if return_lse else out
