"""The paged 8-bit key/value cache: appending to it, selecting its pages, attention over it.

A ``KVCache`` is pages of ``page_size`` tokens for all sequences of a program.  Which page holds the i-th block of tokens of
sequence b says ``table[b, i]``, how many tokens the sequence has ``lengths[b]``, both int32 tensors on the device that the
program keeps; nothing here reads them on the host, so all calls can be captured in a graph and replayed with other lengths.

  cache = cache_create(head_dim, kv_heads, n_pages)
  queries = cache_append(cache, keys, values, table, lengths, queries=queries, rotation=(cos, sin))
  lengths += T
  y = cache_attention(cache, queries, table, lengths)                          # over all pages, or:
  y = cache_attention(cache, queries, table, lengths, pages=cache_select(cache, queries, table, lengths, keep=64))

Tensors of queries, keys and values are ``[B, T, heads * head_dim]``, fp16 or bf16, as those of ``attention_forward``; they may be
slices of a larger tensor as long as the last axis is contiguous and every row starts on a 16-byte boundary.  There is no CPU path,
and there are no gradients: results do not require one, whatever the inputs say.

Tokens are taken back (drafted ones that were not accepted) by lowering ``lengths``.  The pages that they were on keep what they did to
them until a page's first token is appended anew: a scale that they enlarged, the bits that older tokens of the page lost to it, bounds that
still cover them, and a scale that is NaN if one of their values was not finite.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .api import _load_native, _raw_stream

_DTYPES = {torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16}
_CODES = torch.float8_e4m3fn
PAGE_SIZES = (16, 32, 64, 128)

# What the first status word of a cache stands for (fa_cache.cuh).
STATUS = {0: "nothing", 1: "a page outside the cache or the table", 2: "a position or length outside the table or the rotation"}


_native = None   # the extension module's calls, and the library's entries that they go to


def _require(cond: bool, what: str) -> None:
    if not cond:
        raise RuntimeError(f"cache: {what}")


def _calls():
    """(append, select, attention, entries).  A native call answers None for what is not a plain call with every precondition met,
    which then goes through the checks and ctypes below; an int is the status of a launch that failed.  (One token of a short
    sequence on 301 keys: attention 8.1 us a call and 16.9 through ctypes, with the same kernel; append 5.6 and 25.)"""
    global _native
    if _native is None:
        lib = _lib.load()   # raises when the CUDA library is missing: no fallback
        _native = tuple(_load_native(f"_cache_{name}_through") for name in ("append", "select", "attention")) + (lib.cache_entries,)
    return _native


class KVCache:
    """Pages of e4m3 codes with a scale for each page and head, and the bounds of the keys.

    ``k``, ``v``            float8_e4m3fn [n_pages, kv_heads, page_size, head_dim], last axis contiguous, other strides multiples
                            of 16
    ``k_scale``, ``v_scale``  float32 [n_pages, kv_heads], contiguous; a value is code * scale, 2^-100 to 2^120 (one below zero is taken
                            for NaN)
    ``bounds``              float8_e4m3fn [n_pages, kv_heads, 2, head_dim], contiguous: lowest and highest key code

    No code of a token may be NaN (``cache_append`` writes none): in a value it would reach queries that do not see the token.  The tensors are looked at once, here; they must not be moved or resized afterwards.  ``cache_create`` makes them.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, bounds: torch.Tensor):
        for t, name, dtype, dims in ((k, "k", _CODES, 4), (v, "v", _CODES, 4), (k_scale, "k_scale", torch.float32, 2),
                                     (v_scale, "v_scale", torch.float32, 2), (bounds, "bounds", _CODES, 4)):
            _require(isinstance(t, torch.Tensor) and t.dtype == dtype, f"{name} must be a {dtype} tensor")
            _require(t.is_cuda and t.device == k.device, f"{name} must be a CUDA tensor on the device of k")
            _require(t.dim() == dims, f"{name} must have {dims} dimensions")
        n, heads, page, H = k.shape
        _require(H in (16, 32, 64, 128), "head_dim must be 16, 32, 64 or 128")
        _require(page in PAGE_SIZES, "page_size must be 16, 32, 64 or 128")
        _require(n > 0 and heads > 0, "empty tensors are not supported")
        _require(v.shape == k.shape, "v must have the shape of k")
        _require(tuple(k_scale.shape) == (n, heads) and tuple(v_scale.shape) == (n, heads), "scales must have shape [n_pages, kv_heads]")
        _require(tuple(bounds.shape) == (n, heads, 2, H), "bounds must have shape [n_pages, kv_heads, 2, head_dim]")
        _require(k_scale.is_contiguous() and v_scale.is_contiguous() and bounds.is_contiguous(), "scales and bounds must be contiguous")
        for t, name in ((k, "k"), (v, "v")):
            _require(t.stride(3) == 1, f"the last axis of {name} must be contiguous")
            _require(not any(s % 16 for s in t.stride()[:3]), f"the strides of {name} must be multiples of 16")
            _require(max(t.stride()) < 1 << 31 and t.stride(2) <= 1 << 24, f"the strides of {name} must be below 2^31, its tokens' at most 2^24")
        _require(not any(t.data_ptr() % 16 for t in (k, v, bounds)), "k, v and bounds must start on 16-byte boundaries")
        self.k, self.v, self.k_scale, self.v_scale, self.bounds = k, v, k_scale, v_scale, bounds
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = n, heads, page, H
        self.device = k.device
        self._index = k.get_device()
        self._status = torch.zeros(2, dtype=torch.int32, device=k.device)
        self._handle = _lib.Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), bounds.data_ptr(), self._status.data_ptr(),
                                  *k.stride()[:3], *v.stride()[:3], n, heads, page, H)
        self._address = ctypes.addressof(self._handle)
        self._copy_areas = None   # (pages.py)
        # (pages on top of one another can be read, as those of a stand-in for a cache, but not written)
        self._writable = all(t.stride(i) > 0 or t.shape[i] == 1 for t in (k, v) for i in range(3))

    def read_status(self) -> Tuple[int, int]:
        """(first code, number of reports) of what the kernels found wrong in table, lengths, counts or pages; clears it.
        Synchronises.  ``STATUS`` says what the codes mean; 0x100 and above: a bounded wait expired."""
        code, reports = self._status.tolist()
        if code or reports:
            self._status.zero_()
        return code, reports


def cache_create(head_dim: int, kv_heads: int, n_pages: int, page_size: int = 64, device="cuda") -> KVCache:
    """An empty cache."""
    _require(head_dim in (16, 32, 64, 128), "head_dim must be 16, 32, 64 or 128")
    _require(page_size in PAGE_SIZES, "page_size must be 16, 32, 64 or 128")
    _require(n_pages > 0 and kv_heads > 0, "n_pages and kv_heads must be positive")

    def codes(rows: int) -> torch.Tensor:
        return torch.zeros(n_pages, kv_heads, rows, head_dim, dtype=torch.uint8, device=device).view(_CODES)

    def scales() -> torch.Tensor:
        return torch.ones(n_pages, kv_heads, dtype=torch.float32, device=device)
    return KVCache(codes(page_size), codes(page_size), scales(), scales(), codes(2))


def _check_rows(t, name: str, cache: KVCache, B: int, T: int, width: int, dtype) -> None:
    _require(isinstance(t, torch.Tensor) and t.dtype in _DTYPES, f"{name} must be a float16 or bfloat16 tensor")
    _require(dtype is None or t.dtype == dtype, f"{name} must have the type of the others")
    _require(t.get_device() == cache._index and t.is_cuda, f"{name} must be on the cache's device")
    _require(t.dim() == 3, f"{name} must have 3 dimensions")
    _require(B is None or tuple(t.shape[:2]) == (B, T), f"{name} must have shape [B, T, heads * head_dim]")
    _require(t.shape[2] > 0 and t.shape[2] % width == 0 and 0 not in t.shape, f"the last axis of {name} must hold whole heads")
    _require(t.stride(2) == 1, f"the last axis of {name} must be contiguous")
    _require(t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0, f"every row of {name} must start on a 16-byte boundary")


def _sequences(cache: KVCache, table, lengths, counts, B: int, T: int) -> _lib.Sequences:
    for t, name, dims in ((table, "table", 2), (lengths, "lengths", 1)) + (((counts, "counts", 1),) if counts is not None else ()):
        _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32, f"{name} must be an int32 tensor")
        _require(t.is_cuda and t.get_device() == cache._index, f"{name} must be on the cache's device")
        _require(t.dim() == dims and t.shape[0] == B, f"{name} must have {dims} dimension(s), the first of them B")
        _require(t.shape[-1] <= 1 or t.stride(-1) == 1, f"the last axis of {name} must be contiguous")
    _require(table.shape[1] > 0, "the table has no pages")
    return _lib.Sequences(table.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr(), table.stride(0), table.shape[1], B, T)


def cache_append(cache: KVCache, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                 counts: Optional[torch.Tensor] = None, queries: Optional[torch.Tensor] = None,
                 rotation: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write T new tokens of each sequence into its pages, behind the ``lengths[b]`` tokens that it holds.

    ``keys``, ``values``  [B, T, kv_heads * head_dim];  ``table`` int32 [B, W];  ``lengths`` int32 [B], not changed
    ``counts``    int32 [B]: how many of the T tokens sequence b has (default: all)
    ``queries``   [B, T, heads * head_dim]: rotated like the keys and returned as a new tensor, zeros where there is no token
    ``rotation``  (cos, sin), float32 [positions, head_dim / 2] each: keys and queries are rotated by their position, pairs of
                  dimensions (i, i + head_dim / 2), or (2 i, 2 i + 1) with ``interleaved``; tokens behind the last position are
                  not appended, their queries come back as zeros, and ``read_status`` tells

    Each page keeps, by head, one power of two as the scale of its keys and one as that of its values, such that the largest
    magnitude comes to lie in the upper half of e4m3's range; where a later token needs a larger scale the page's codes move to it.
    Two sequences must not append to the same page in one call (they may share full pages).
    """
    _require(isinstance(cache, KVCache), "the first argument must be a KVCache")
    append, _, _, entries = _calls()
    if cache._writable:
        done = append(entries[0], cache._address, cache._index, keys, values, table, lengths, counts, queries, rotation, interleaved)
        if done is not None:
            if done.__class__ is int:
                _lib.check(done)
            return None if done is True else done
    _check_rows(keys, "keys", cache, None, None, cache.head_dim, None)
    B, T, F = keys.shape
    _require(F == cache.kv_heads * cache.head_dim, "keys must have kv_heads * head_dim features")
    _check_rows(values, "values", cache, B, T, F, keys.dtype)
    _require(values.shape == keys.shape, "values must have the shape of keys")
    _require(cache._writable, "the pages of this cache lie on top of one another: it cannot be appended to")
    sequences = _sequences(cache, table, lengths, counts, B, T)
    rotated = q = None
    q_strides, heads = (0, 0), 0
    if queries is not None:
        _check_rows(queries, "queries", cache, B, T, cache.head_dim, keys.dtype)
        heads = queries.shape[2] // cache.head_dim
        rotated = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device)
        q, q_strides = queries.data_ptr(), queries.stride()
    cos = sin = None
    positions = 0
    if rotation is not None:
        _require(isinstance(rotation, (tuple, list)) and len(rotation) == 2, "rotation must be (cos, sin)")
        cos, sin = rotation
        for t, name in ((cos, "cos"), (sin, "sin")):
            _require(isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.is_cuda and t.get_device() == cache._index,
                     f"{name} must be a float32 tensor on the cache's device")
            _require(t.dim() == 2 and t.shape[1] == cache.head_dim // 2 and t.shape == cos.shape and t.shape[0] > 0 and t.is_contiguous()
                     and t.data_ptr() % 16 == 0, f"{name} must be contiguous, of shape [positions, head_dim / 2], on a 16-byte boundary")
        positions = min(cos.shape[0], 0x7FFFFFFF)
        cos, sin = cos.data_ptr(), sin.data_ptr()
    _lib.check(_lib.load().fa_b200_cache_append(
        ctypes.byref(cache._handle), ctypes.byref(sequences), keys.data_ptr(), keys.stride(0), keys.stride(1), values.data_ptr(), values.stride(0),
        values.stride(1), q, q_strides[0], q_strides[1], heads, None if rotated is None else rotated.data_ptr(), cos, sin, positions,
        _DTYPES[keys.dtype], _lib.CACHE_NEIGHBOURS if interleaved else 0, cache._index, _raw_stream(cache._index)))
    return rotated


def cache_select(cache: KVCache, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, keep: int, *,
                 counts: Optional[torch.Tensor] = None, first: int = 1, last: int = 1) -> torch.Tensor:
    """The ``keep`` pages that each query and key/value head should attend to: int32 [B, T, kv_heads, keep], ascending block
    indices of the sequence, -1 behind the last.

    Among the pages up to the query's own those are taken whose keys, by the page's bounds, may have the largest product with the
    query (for query heads that share a key/value head the largest of theirs), the lower page where two are equal; the ``first`` first
    and the ``last`` last ones in any case, before all others.  ``queries`` (rotated), ``table``, ``lengths`` and ``counts`` as
    for ``cache_attention``.  Queries are rounded to 8 bits for this and bounds to multiples of four codes, to nearest, so that a score is
    an estimate of the bound and not one itself.  Of the 64 best of 1000 pages of normal keys by the bounds as they are, 99.6 % are found;
    with four dimensions 20 times as large as the others, beside which theirs become few multiples, 84 %.
    """
    _require(isinstance(cache, KVCache), "the first argument must be a KVCache")
    _, select, _, entries = _calls()
    pages = select(entries[1], cache._address, cache._index, queries, table, lengths, counts, keep, first, last)
    if pages is not None:
        if pages.__class__ is int:
            _lib.check(pages)
        return pages
    _check_rows(queries, "queries", cache, None, None, cache.kv_heads * cache.head_dim, None)
    B, T, F = queries.shape
    sequences = _sequences(cache, table, lengths, counts, B, T)
    _require(1 <= keep <= 0x7FFFFFFF, "keep must be positive")
    _require(first >= 0 and last >= 1, "first must not be negative, last at least 1")
    pages = torch.empty(B, T, cache.kv_heads, keep, dtype=torch.int32, device=cache.device)
    scratch = torch.empty(B * T * cache.kv_heads * table.shape[1], dtype=torch.int32, device=cache.device)
    _lib.check(_lib.load().fa_b200_cache_select(
        ctypes.byref(cache._handle), ctypes.byref(sequences), queries.data_ptr(), queries.stride(0), queries.stride(1), F // cache.head_dim,
        _DTYPES[queries.dtype], keep, min(first, 0x7FFFFFFF), min(last, 0x7FFFFFFF), pages.data_ptr(), scratch.data_ptr(), 4 * scratch.numel(), cache._index,
        _raw_stream(cache._index)))
    return pages


@lru_cache(maxsize=4096)
def _scratch_bytes(head_dim: int, kv_heads: int, heads: int, page: int, B: int, T: int, width: int, keep: int, device: int) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.load().fa_b200_cache_attention_scratch(head_dim, kv_heads, heads, page, B, T, width, keep, device, ctypes.byref(out)))
    return out.value


def cache_attention(cache: KVCache, queries: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                    counts: Optional[torch.Tensor] = None, pages: Optional[torch.Tensor] = None, causal: bool = True,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(Q K^T / sqrt(head_dim)) V`` of T queries a sequence over the cache, [B, T, heads * head_dim] of the queries' type.

    The queries are the last tokens of their sequences: query t stands at position ``lengths[b] - T + t`` (``lengths[b] -
    counts[b] + t`` where ``counts`` says how many of the T a sequence has) and sees the keys up to its own; with ``causal=False``
    all keys of its sequence.  ``heads`` is a multiple of the cache's kv_heads, query head h goes with key/value head
    h // (heads // kv_heads).  ``pages`` int32 [B, T, kv_heads, keep], as ``cache_select`` returns it: only these blocks of the
    sequence, each at most once, -1 for nothing.  A query that sees no key, or that its sequence does not have, gets zeros.

    Scores and sums are held in 32 bits.  The weights are rounded to fp16 for their product with the values; with fewer than 64 rows (T *
    heads / kv_heads), or with ``pages``, fp16 calls multiply what that loses too: their error is little more than the result's rounding.
    """
    _require(isinstance(cache, KVCache), "the first argument must be a KVCache")
    _, _, attention, entries = _calls()
    y = attention(entries[2], entries[3], cache._address, cache._index, queries, table, lengths, counts, pages, causal, out)
    if y is not None:
        if y.__class__ is int:
            _lib.check(y)
        return y
    _check_rows(queries, "queries", cache, None, None, cache.kv_heads * cache.head_dim, None)
    B, T, F = queries.shape
    sequences = _sequences(cache, table, lengths, counts, B, T)
    keep = 0
    if pages is not None:
        _require(isinstance(pages, torch.Tensor) and pages.dtype == torch.int32 and pages.is_cuda and pages.get_device() == cache._index,
                 "pages must be an int32 tensor on the cache's device")
        _require(pages.dim() == 4 and tuple(pages.shape[:3]) == (B, T, cache.kv_heads) and pages.shape[3] > 0 and pages.is_contiguous(),
                 "pages must be contiguous, of shape [B, T, kv_heads, keep]")
        keep = pages.shape[3]
    if out is None:
        out = torch.empty((B, T, F), dtype=queries.dtype, device=cache.device)
    else:
        _require(isinstance(out, torch.Tensor) and out.dtype == queries.dtype and out.is_cuda and out.get_device() == cache._index
                 and tuple(out.shape) == (B, T, F) and out.is_contiguous() and out.data_ptr() % 16 == 0, "out must match queries and be contiguous")
    heads = F // cache.head_dim
    scratch = torch.empty(_scratch_bytes(cache.head_dim, cache.kv_heads, heads, cache.page_size, B, T, table.shape[1], keep, cache._index),
                          dtype=torch.uint8, device=cache.device)
    _lib.check(_lib.load().fa_b200_cache_attention(
        ctypes.byref(cache._handle), ctypes.byref(sequences), queries.data_ptr(), queries.stride(0), queries.stride(1), heads, _DTYPES[queries.dtype],
        None if pages is None else pages.data_ptr(), keep, 0 if causal else _lib.CACHE_ALL_KEYS, out.data_ptr(), scratch.data_ptr(), scratch.numel(),
        cache._index, _raw_stream(cache._index)))
    return out
