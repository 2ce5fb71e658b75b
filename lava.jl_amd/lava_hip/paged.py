"""A paged key/value cache and the attention of new tokens over it: `kv_append`, `paged_attn` and
`shared_prefix_attn`, destination-first like the other kernels, over HIPDeviceArrays or raw device addresses.

Arrays keep the attention's order, head dimension fastest: a cache is an (E, L, H, P) array of P pages of L
tokens, a batch's queries, keys and values are (E, H, T) arrays of the T new tokens of all its sequences, one
sequence behind the other (`q_start`).  The `*_raw` constructors make the descriptors of include/lava_hip.h
from addresses; a serving program makes them once and fills new lengths and tables into the device arrays that
they name.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

from . import _lib
from .device import DTYPES, HIPDeviceArray, synchronize


def _fits(bits: int, **values: int) -> None:
    """Refuses what a descriptor's integers would cut off."""
    for name, x in values.items():
        if not -2 ** (bits - 1) <= x < 2 ** (bits - 1):
            raise ValueError(f"{name} = {x} does not fit {bits} bits")


def _fits_size(**values: int) -> None:
    """Refuses a number of bytes that a size_t would cut off, or take a negative one for the largest there is."""
    for name, x in values.items():
        if not 0 <= x < 2 ** 64:
            raise ValueError(f"{name} = {x} is no size")


def paged_cache_raw(dtype: str, k: int, v: int, head_dim: int, page_size: int, heads: int, pages: int,
                    strides: Sequence[int]) -> _lib.KVCacheDesc:
    """Pages of keys at `k` and of values at `v`, both with element strides of (E, L, H, P)."""
    if dtype not in DTYPES:
        raise ValueError(f"unknown element type {dtype!r}; one of {sorted(DTYPES)}")
    _fits(32, head_dim=head_dim, page_size=page_size, heads=heads)
    _fits(64, pages=pages, **{f"strides[{i}]": st for i, st in enumerate(strides)})
    return _lib.KVCacheDesc(k, v, DTYPES[dtype][0], head_dim, page_size, heads, pages, (C.c_int64 * 4)(*strides))


def paged_batch_raw(sequences: int, tokens: int, q_start: int, kv_len: int, table: int, max_pages: int,
                    max_q: int = 0, workspace: int = 0, workspace_bytes: int = 0) -> _lib.KVBatchDesc:
    """A ragged batch by the addresses of its int32 q_start (B + 1), kv_len (B) and page table (B rows of
    max_pages)."""
    _fits(32, sequences=sequences, max_pages=max_pages)
    _fits(64, tokens=tokens, max_q=max_q)
    _fits_size(workspace_bytes=workspace_bytes)
    return _lib.KVBatchDesc(sequences, max_pages, tokens, max_q, q_start, kv_len, table, workspace or None,
                            workspace_bytes)


def rope_raw(inv_freq: int, rot_dim: int, interleaved: bool = False, positions: int = 0,
             offset: int = 0) -> _lib.RopeDesc:
    _fits(32, rot_dim=rot_dim, offset=offset)
    return _lib.RopeDesc(inv_freq or None, rot_dim, int(bool(interleaved)), positions or None, offset)


def attn_score_raw(scale: float, causal: bool = True, window: int = 0, cap: float = 0.0, slopes: int = 0,
                   bidirectional: int = 0) -> _lib.AttnScoreDesc:
    _fits(32, window=window)
    return _lib.AttnScoreDesc(scale, cap, int(bool(causal)), window, slopes or None, bidirectional or None)


_I64x3 = C.c_int64 * 3


def _strides(st: Optional[Sequence[int]]):
    return _I64x3(*st) if st is not None else None


def kv_append_raw(cache: _lib.KVCacheDesc, batch: _lib.KVBatchDesc, K: int, V: int, kv_strides: Sequence[int],
                  Q: int = 0, Q_out: int = 0, q_heads: int = 0, q_strides: Optional[Sequence[int]] = None,
                  qo_strides: Optional[Sequence[int]] = None, rope: Optional[_lib.RopeDesc] = None,
                  stream: Optional[int] = None) -> None:
    """The new tokens' K and V into the cache, K (and Q into Q_out) turned by `rope`; strides of (E, H, T)."""
    _lib.call("lava_hip_kv_append", C.byref(cache), C.byref(batch), K, V, _strides(kv_strides), Q or None, Q_out or None,
              q_heads, _strides(q_strides), _strides(qo_strides), C.byref(rope) if rope is not None else None, stream)


def paged_attn_raw(cache: _lib.KVCacheDesc, batch: _lib.KVBatchDesc, score: _lib.AttnScoreDesc, Q: int, O: int,
                   q_heads: int, q_strides: Sequence[int], o_strides: Sequence[int], lse: int = 0,
                   stream: Optional[int] = None) -> None:
    _lib.call("lava_hip_paged_attn", C.byref(cache), C.byref(batch), C.byref(score), Q, O, q_heads, _strides(q_strides),
              _strides(o_strides), lse or None, stream)


def shared_prefix_attn_raw(cache: _lib.KVCacheDesc, batch: _lib.KVBatchDesc, score: _lib.AttnScoreDesc,
                           prefix_pages: int, prefix_len: int, Q: int, O: int, q_heads: int, q_strides: Sequence[int],
                           o_strides: Sequence[int], lse: int = 0, stream: Optional[int] = None) -> None:
    _lib.call("lava_hip_shared_prefix_attn", C.byref(cache), C.byref(batch), C.byref(score), prefix_pages or None,
              prefix_len, Q, O, q_heads, _strides(q_strides), _strides(o_strides), lse or None, stream)


def paged_workspace_bytes(cache: _lib.KVCacheDesc, batch: _lib.KVBatchDesc, q_heads: int, prefix_len: int = 0) -> int:
    """Bytes of workspace for attention calls with these descriptors (`paged_batch_raw(..., workspace=)`)."""
    n = C.c_size_t()
    _lib.call("lava_hip_paged_workspace_bytes", C.byref(cache), C.byref(batch), q_heads, prefix_len, C.byref(n))
    return int(n.value)


class PagedCache:
    """A cache of `pages` pages of `page_size` tokens: (E, L, H, P) arrays `k` and `v`."""

    def __init__(self, dtype: str, head_dim: int, page_size: int, heads: int, pages: int):
        self.k = HIPDeviceArray(dtype, (head_dim, page_size, heads, pages))
        self.v = HIPDeviceArray(dtype, (head_dim, page_size, heads, pages))
        self.dtype, self.head_dim, self.page_size, self.heads, self.pages = dtype, head_dim, page_size, heads, pages
        self.desc = paged_cache_raw(dtype, self.k.ptr, self.v.ptr, head_dim, page_size, heads, pages, self.k.strides())

    def close(self) -> None:
        self.k.close()
        self.v.close()


class PagedBatch:
    """The lengths and page tables of a ragged batch, int32 device arrays: q_start (B + 1), kv_len (B), table
    (max_pages, B).  `tokens` is the T of its (E, H, T) arrays, max_q the most new tokens of a sequence (0: unknown)."""

    def __init__(self, tokens: int, q_start: HIPDeviceArray, kv_len: HIPDeviceArray, table: HIPDeviceArray,
                 max_q: int = 0):
        for a in (q_start, kv_len, table):
            if a.dtype != "i32":
                raise ValueError(f"q_start, kv_len and table are i32 arrays (got {a.dtype})")
        if len(table.dims) != 2 or table.order != "F":
            raise ValueError("table must be a column-major (max_pages, B) array")
        B = table.dims[1]
        if q_start.size != B + 1 or kv_len.size != B:
            raise ValueError(f"shape mismatch: q_start {q_start.dims}, kv_len {kv_len.dims}, table {table.dims}")
        self.q_start, self.kv_len, self.table = q_start, kv_len, table
        self.tokens = tokens
        self.workspace: Optional[HIPDeviceArray] = None
        self.desc = paged_batch_raw(B, tokens, q_start.ptr, kv_len.ptr, table.ptr, table.dims[0], max_q)

    def own_workspace(self, cache: PagedCache, q_heads: int, prefix_len: int = 0) -> "PagedBatch":
        """Gives the batch's attention calls a workspace of its own in place of the stream's (allocated here, so before a
        capture): for calls that may run at once with others of their stream's, such as replayed graphs."""
        ws = HIPDeviceArray("u8", (paged_workspace_bytes(cache.desc, self.desc, q_heads, prefix_len),))
        ws.fill_bytes(0)
        synchronize()   # whatever stream the calls are on
        self.workspace = ws
        self.desc.workspace, self.desc.workspace_bytes = ws.ptr or None, ws.nbytes
        return self


def _check_tokens(name: str, a: HIPDeviceArray, cache: PagedCache, batch: PagedBatch) -> None:
    if a.dtype != cache.dtype or len(a.dims) != 3 or a.order != "F":
        raise ValueError(f"{name} must be a column-major 3-D {cache.dtype} array (E, H, T)")
    if a.dims[0] != cache.head_dim or a.dims[2] != batch.tokens:
        raise ValueError(f"shape mismatch: {name} {a.dims}, head dimension {cache.head_dim}, {batch.tokens} tokens")


def kv_append(cache: PagedCache, batch: PagedBatch, K: HIPDeviceArray, V: HIPDeviceArray,
              Q: Optional[HIPDeviceArray] = None, Q_out: Optional[HIPDeviceArray] = None,
              inv_freq: Optional[HIPDeviceArray] = None, interleaved: bool = False,
              positions: Optional[HIPDeviceArray] = None, offset: int = 0, stream: Optional[int] = None) -> PagedCache:
    """Appends the batch's new K and V, (E, H, T) arrays, to the cache.  With `inv_freq` (f32, half the rotated
    elements) K, and Q into Q_out (default: in place), turn by their tokens' positions: `positions` (i32, T) or
    offset + the place in the sequence."""
    for name, a in (("K", K), ("V", V)):
        _check_tokens(name, a, cache, batch)
        if a.dims[1] != cache.heads:
            raise ValueError(f"{name} has {a.dims[1]} heads, the cache {cache.heads}")
    if Q is None and Q_out is not None:
        raise ValueError("Q_out without Q")
    if Q is not None:
        Q_out = Q if Q_out is None else Q_out
        _check_tokens("Q", Q, cache, batch)
        if Q_out.dtype != Q.dtype or Q_out.dims != Q.dims or Q_out.order != "F":
            raise ValueError("Q_out must be like Q")
    rope = None
    if inv_freq is not None:
        if inv_freq.dtype != "f32":
            raise ValueError(f"inv_freq must be f32 (got {inv_freq.dtype})")
        if positions is not None and (positions.dtype != "i32" or positions.size != batch.tokens):
            raise ValueError("positions must be an i32 vector, one per token")
        rope = rope_raw(inv_freq.ptr, 2 * inv_freq.size, interleaved, positions.ptr if positions is not None else 0,
                        offset)
    kv_append_raw(cache.desc, batch.desc, K.ptr, V.ptr, K.strides(), Q.ptr if Q is not None else 0,
                  Q_out.ptr if Q is not None else 0, Q.dims[1] if Q is not None else 0,
                  Q.strides() if Q is not None else None, Q_out.strides() if Q is not None else None, rope, stream)
    return cache


def _attn_args(O, cache, batch, Q, scale, causal, window, cap, slopes, bidirectional, lse):
    _check_tokens("Q", Q, cache, batch)
    _check_tokens("O", O, cache, batch)
    Hq = Q.dims[1]
    if O.dims != Q.dims:
        raise ValueError(f"shape mismatch: O {O.dims}, Q {Q.dims}")
    if slopes is not None and (slopes.dtype != "f32" or slopes.size != Hq):
        raise ValueError("slopes must be an f32 vector, one per query head")
    if bidirectional is not None and (bidirectional.dtype != "i32" or bidirectional.size != batch.kv_len.size):
        raise ValueError("bidirectional must be an i32 vector, one per sequence")
    if lse is not None and (lse.dtype != "f32" or lse.dims != (Hq, batch.tokens) or lse.order != "F"):
        raise ValueError("lse must be a column-major (H, T) f32 array")
    sc = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    score = attn_score_raw(sc, causal, window, cap, slopes.ptr if slopes is not None else 0,
                           bidirectional.ptr if bidirectional is not None else 0)
    return score, Hq, lse.ptr if lse is not None else 0


def paged_attn(O: HIPDeviceArray, cache: PagedCache, batch: PagedBatch, Q: HIPDeviceArray,
               scale: Optional[float] = None, causal: bool = True, window: int = 0, cap: float = 0.0,
               slopes: Optional[HIPDeviceArray] = None, bidirectional: Optional[HIPDeviceArray] = None,
               lse: Optional[HIPDeviceArray] = None, stream: Optional[int] = None) -> HIPDeviceArray:
    """O = softmax(scores of the new tokens' queries with their sequences' cached keys) times the cached values,
    (E, H, T) arrays; the scores' scale, cap, distance slopes and masks are those of `lava_hip_attn_score`."""
    score, Hq, lp = _attn_args(O, cache, batch, Q, scale, causal, window, cap, slopes, bidirectional, lse)
    paged_attn_raw(cache.desc, batch.desc, score, Q.ptr, O.ptr, Hq, Q.strides(), O.strides(), lp, stream)
    return O


def shared_prefix_attn(O: HIPDeviceArray, cache: PagedCache, batch: PagedBatch, prefix_pages: HIPDeviceArray,
                       prefix_len: int, Q: HIPDeviceArray, scale: Optional[float] = None, causal: bool = True,
                       window: int = 0, cap: float = 0.0, slopes: Optional[HIPDeviceArray] = None,
                       lse: Optional[HIPDeviceArray] = None, stream: Optional[int] = None) -> HIPDeviceArray:
    """`paged_attn` for sequences that all begin with the prefix_len tokens in `prefix_pages` (i32): the batch's
    lengths and tables are those of each sequence's own tokens behind it."""
    if prefix_pages.dtype != "i32" or prefix_pages.size * cache.page_size < prefix_len:
        raise ValueError(f"prefix_pages must be i32 pages of at least {prefix_len} tokens")
    score, Hq, lp = _attn_args(O, cache, batch, Q, scale, causal, window, cap, slopes, None, lse)
    shared_prefix_attn_raw(cache.desc, batch.desc, score, prefix_pages.ptr, prefix_len, Q.ptr, O.ptr, Hq, Q.strides(),
                           O.strides(), lp, stream)
    return O
