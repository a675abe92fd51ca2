"""A paged cache of keys and values, Gaussian moments in float32, bfloat16 or 8 bits.

Four pools, means and variances of keys and values, each (pages, heads, page_size, head_dim). In
8 bits (e4m3) a row of head_dim holds codes and one power of two: the least with
max|x| <= 448 * 2^e; ``scales`` (pages, heads, page_size, 4) holds e + 127 of a row's key means,
key variances, value means and value variances. Values are rounded to the nearest, ties to even.

A sequence's tokens lie in the pages that its row of ``table`` (B, width) int32 names, in order:
token n in page table[b, n // page_size]. Tokens whose page is not in the table, or outside the
pool, do not exist: they are not written, read as zeros, and attention does not see them. (Page
numbers are on the GPU; raising an error for them would wait for it.)
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .. import _lib
from ._operands import counts as counts_of, heads as heads_of, pair, shape_of

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}


class KVCache(NamedTuple):
    """The pools of a cache: any tensors of the shapes above; ``new_kv_cache`` makes them."""

    km: Tensor
    kS: Tensor
    vm: Tensor
    vS: Tensor
    scales: Tensor | None = None


def new_kv_cache(pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.float32,
                 device="cuda") -> KVCache:
    if dtype not in _TYPES:
        raise TypeError(f"KVCache holds float32, bfloat16 or float8_e4m3fn, got {dtype}")
    if min(pages, heads, page_size, head_dim) < 1:
        raise ValueError(f"bad sizes: {pages} pages, {heads} heads, {page_size} tokens, {head_dim} features")
    shape = (pages, heads, page_size, head_dim)
    pools = [torch.zeros(shape, device=device, dtype=torch.uint8 if dtype is torch.float8_e4m3fn else dtype)
             for _ in range(4)]
    if dtype is not torch.float8_e4m3fn:
        return KVCache(*pools)
    scales = torch.ones((*shape[:3], 4), device=device, dtype=torch.uint8)
    return KVCache(*(p.view(dtype) for p in pools), scales)


def cache_struct(cache: KVCache, ref: Tensor) -> _lib.KvCache:
    """The library's description of a cache on ref's GPU."""
    if not isinstance(cache, KVCache):
        raise TypeError(f"cache: expected a KVCache, got {type(cache).__name__}")
    km, kS, vm, vS, scales = cache
    shape, dtype, dev = km.shape, km.dtype, ref.get_device()
    kind = _TYPES.get(dtype)
    if kind is None:
        raise TypeError(f"cache: holds float32, bfloat16 or float8_e4m3fn, got {dtype}")
    if len(shape) != 4 or 0 in shape[1:]:
        raise ValueError(f"cache: expected (pages, heads, page_size, head_dim), got {tuple(shape)}")
    if shape[3] > 128:
        raise ValueError(f"cache: head dimensions up to 128, got {shape[3]}")
    for t, n in ((km, "km"), (kS, "kS"), (vm, "vm"), (vS, "vS")):
        if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"cache {n}: expected contiguous {dtype} {tuple(shape)} on {ref.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if kind == 2:
        if (not isinstance(scales, Tensor) or scales.dtype is not torch.uint8 or scales.get_device() != dev
                or tuple(scales.shape) != (*shape[:3], 4) or not scales.is_contiguous()):
            raise ValueError(f"cache scales: expected contiguous uint8 {(*shape[:3], 4)} on {ref.device}")
    return _lib.KvCache(km.data_ptr(), kS.data_ptr(), vm.data_ptr(), vS.data_ptr(),
                        scales.data_ptr() if kind == 2 else None, kind, *shape)


def check_table(table: Tensor, ref: Tensor, B: int) -> Tensor:
    if not isinstance(table, Tensor) or table.dtype is not torch.int32:
        raise TypeError("table: expected an int32 tensor")
    if table.device != ref.device or table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table: expected ({B}, pages of a sequence) on {ref.device}, got {tuple(table.shape)} on "
                         f"{table.device}")
    return table.contiguous()


def cache_write(cache: KVCache, mk: Tensor, Sk: Tensor, mv: Tensor, Sv: Tensor, table: Tensor,
                starts: Tensor | None = None, counts: Tensor | None = None) -> None:
    """Tokens t < ``counts[b]`` (all without) of keys and values (B, T, heads, head_dim) become tokens
    ``starts[b]`` + t (t without) of the cache. Pages that get tokens are named once in ``table``."""
    shape = shape_of(mk, "mk", 4)
    B, T, G, D = shape
    mk, Sk = pair(mk, Sk, "k", mk, shape)
    mv, Sv = pair(mv, Sv, "v", mk, shape)
    c = cache_struct(cache, mk)
    if (c.heads, c.head_dim) != (G, D):
        raise ValueError(f"cache: holds {c.heads} heads of {c.head_dim}, got {G} of {D}")
    table = check_table(table, mk, B)
    starts, start_bytes = counts_of(starts, "starts", mk, B)
    counts, count_bytes = counts_of(counts, "counts", mk, B)
    _lib.call_on(mk, "tagi_kv_cache_write", c, mk.data_ptr(), Sk.data_ptr(), heads_of(mk), mv.data_ptr(), Sv.data_ptr(),
                 heads_of(mv), table.data_ptr(), table.shape[1], _lib.ptr(starts), start_bytes, _lib.ptr(counts),
                 count_bytes, B, T, _lib.stream_of(mk))


def cache_read(cache: KVCache, table: Tensor, lengths: Tensor, tokens: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(mk, Sk, mv, Sv) of tokens n < ``tokens`` of every sequence, (B, tokens, heads, head_dim) float32;
    zeros from ``lengths[b]`` on."""
    if not isinstance(table, Tensor) or not table.is_cuda:
        raise ValueError("table: the TAGI HIP kernels run on the GPU only")
    c = cache_struct(cache, table)
    B = table.shape[0]
    table = check_table(table, table, B)
    if lengths is None:
        raise TypeError("lengths: expected an int32 or int64 tensor")
    lengths, len_bytes = counts_of(lengths, "lengths", table, B)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    mk = torch.empty((B, tokens, c.heads, c.head_dim), device=table.device, dtype=torch.float32)
    out = (mk, *(torch.empty_like(mk) for _ in range(3)))
    _lib.call_on(table, "tagi_kv_cache_read", c, table.data_ptr(), table.shape[1], lengths.data_ptr(), len_bytes,
                 *(t.data_ptr() for t in out), B, tokens, _lib.stream_of(table))
    return out
