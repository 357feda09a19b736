"""The paged cache of latent vectors: one row a token for all heads, appending to it, attention over it.

A token's row holds ``latent_dim`` 16-bit values that are key and value at once, and ``rope_dim`` more that are rotated by the token's position
and belong to the key alone.  Tables, lengths and counts are those of the 8-bit cache (cache.py), pages are managed alike (pages.py).

  cache = latent_cache_create(latent_dim=512, rope_dim=64, n_pages=4096)                  # one per layer
  keys, q_rope = latent_append(cache, latents, rope_keys, table, lengths, queries=q_rope, rotation=(cos, sin))
  lengths += T
  y = latent_attention(cache, q_latent, q_rope, table, lengths, scale=(nope + rope) ** -0.5)   # queries multiplied into the latent space

``latent_attention`` is the absorbed form: with keys W_k c and values W_v c of a head, its queries are q_latent = W_k^T q, and its
results still have to be multiplied by W_v.  It reads a token once for all heads, which is what single tokens need; for a prompt
``latent_prompt`` takes the keys and values multiplied out, with a third of the products.

Tensors are fp16 or bf16, of the cache's type, ``[B, T, dim]`` or ``[B, T, heads, dim]``; they may be slices of larger ones as long as the last
axis is contiguous and every row starts on a 16-byte boundary.  There is no CPU path, and there are no gradients.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .api import _load_native, _raw_stream
from .cache import PAGE_SIZES

_DTYPES = {torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16}
LATENT_DIMS, ROPE_DIMS = (128, 256, 512), (16, 32, 64)


_native = None   # the extension module's calls, and the library's entries that they go to


def _require(cond: bool, what: str) -> None:
    if not cond:
        raise RuntimeError(f"latent: {what}")


def _calls():
    """(append, attention, prompt, entries): as in cache.py, None is the answer to what goes through the checks and ctypes below, an int the
    status of a launch that failed."""
    global _native
    if _native is None:
        lib = _lib.load()   # raises when the CUDA library is missing: no fallback
        _native = tuple(_load_native(f"_latent_{name}_through") for name in ("append", "attention", "prompt")) + (lib.latent_entries,)
    return _native


class LatentCache:
    """Pages of latent vectors: ``data``, fp16 or bf16 [n_pages, page_size, latent_dim + rope_dim], last axis contiguous, other strides multiples
    of 8.  The tensor is looked at once, here; it must not be moved or resized afterwards.  ``latent_cache_create`` makes it."""

    def __init__(self, data: torch.Tensor, latent_dim: int):
        _require(isinstance(data, torch.Tensor) and data.dtype in _DTYPES, "data must be a float16 or bfloat16 tensor")
        _require(data.is_cuda, "data must be a CUDA tensor")
        _require(data.dim() == 3 and 0 not in data.shape and data.shape[0] < 0x7FFFFFFF, "data must have shape [n_pages, page_size, latent_dim + rope_dim]")
        n, page, width = data.shape
        _require(latent_dim in LATENT_DIMS, "latent_dim must be 128, 256 or 512")
        _require(width - latent_dim in ROPE_DIMS, "rope_dim must be 16, 32 or 64")
        _require(page in PAGE_SIZES, "page_size must be 16, 32, 64 or 128")
        _require(data.stride(2) == 1, "the last axis of data must be contiguous")
        _require(all(s % 8 == 0 and s > 0 for s in data.stride()[:2]), "the strides of data must be positive multiples of 8")
        _require(data.stride(0) < 1 << 30 and data.stride(1) <= 1 << 23, "the strides of data must be below 2^30, its tokens' at most 2^23")
        _require(data.data_ptr() % 16 == 0, "data must start on a 16-byte boundary")
        self.data, self.n_pages, self.page_size, self.latent_dim, self.rope_dim = data, n, page, latent_dim, width - latent_dim
        self.dtype, self.device, self._index, self._code = data.dtype, data.device, data.get_device(), _DTYPES[data.dtype]
        self._status = torch.zeros(2, dtype=torch.int32, device=data.device)
        self._handle = _lib.LatentCache(data.data_ptr(), self._status.data_ptr(), 2 * data.stride(0), 2 * data.stride(1), n, page, latent_dim, self.rope_dim)
        self._address = ctypes.addressof(self._handle)
        self._copy_areas = None
        # (rows on top of one another can be read, but not written; pages may lie among one another's tokens)
        reach, self._writable = width, True
        for stride, size in sorted((data.stride(i), data.shape[i]) for i in range(2) if data.shape[i] > 1):
            self._writable = self._writable and stride >= reach
            reach += stride * (size - 1)

    def read_status(self) -> Tuple[int, int]:
        """(first code, number of reports) of what the kernels found wrong in table and lengths; clears it.  Synchronises.  The codes are those of
        ``cache.STATUS``; 0x100 and above: a bounded wait expired.  (Counts are cut to 0 to T and not reported.)"""
        code, reports = self._status.tolist()
        if code or reports:
            self._status.zero_()
        return code, reports


def latent_cache_create(latent_dim: int, rope_dim: int, n_pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda") -> LatentCache:
    """An empty cache."""
    _require(latent_dim in LATENT_DIMS, "latent_dim must be 128, 256 or 512")
    _require(rope_dim in ROPE_DIMS, "rope_dim must be 16, 32 or 64")
    _require(page_size in PAGE_SIZES, "page_size must be 16, 32, 64 or 128")
    _require(n_pages > 0, "n_pages must be positive")
    _require(dtype in _DTYPES, "dtype must be float16 or bfloat16")
    return LatentCache(torch.zeros(n_pages, page_size, latent_dim + rope_dim, dtype=dtype, device=device), latent_dim)


def _check_rows(t, name: str, dtype, index: int, shape) -> None:
    """``shape``: sizes, None where any will do."""
    _require(isinstance(t, torch.Tensor) and t.dtype in _DTYPES, f"{name} must be a float16 or bfloat16 tensor")
    _require(dtype is None or t.dtype == dtype, f"{name} must have the type of the others")
    _require(t.is_cuda and (index is None or t.get_device() == index), f"{name} must be a CUDA tensor on the device of the others")
    _require(t.dim() == len(shape) and 0 not in t.shape and all(n is None or t.shape[i] == n for i, n in enumerate(shape)),
             f"{name} must have shape [{', '.join('*' if n is None else str(n) for n in shape)}], with no axis empty")
    _require(t.stride(-1) == 1, f"the last axis of {name} must be contiguous")
    _require(t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1), f"every row of {name} must start on a 16-byte boundary")


def _strides(t: torch.Tensor):
    """Of all axes but the last; an axis of one is nowhere stepped along."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape))


def _sequences(cache: LatentCache, table, lengths, counts, B: int, T: int) -> _lib.Sequences:
    for t, name, dims in ((table, "table", 2), (lengths, "lengths", 1)) + (((counts, "counts", 1),) if counts is not None else ()):
        _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32, f"{name} must be an int32 tensor")
        _require(t.is_cuda and t.get_device() == cache._index, f"{name} must be on the cache's device")
        _require(t.dim() == dims and t.shape[0] == B, f"{name} must have {dims} dimension(s), the first of them B")
        _require(t.shape[-1] <= 1 or t.stride(-1) == 1, f"the last axis of {name} must be contiguous")
    _require(table.shape[1] > 0, "the table has no pages")
    return _lib.Sequences(table.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr(), table.stride(0), table.shape[1], B, T)


def latent_append(cache: LatentCache, latents: torch.Tensor, rope_keys: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                  counts: Optional[torch.Tensor] = None, queries: Optional[torch.Tensor] = None, rotation: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                  interleaved: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Write T new tokens of each sequence into its pages, behind the ``lengths[b]`` tokens that it holds; (rotated keys, rotated queries).

    ``latents``    [B, T, latent_dim], written as they are;  ``rope_keys`` [B, T, rope_dim], rotated by their position on the way
    ``table`` int32 [B, W];  ``lengths`` int32 [B], not changed;  ``counts`` int32 [B]: how many of the T tokens sequence b has (default: all)
    ``queries``    [B, T, heads, rope_dim]: the rotary part of the queries, rotated like the keys (None: none are returned)
    ``rotation``   (cos, sin), float32 [positions, rope_dim / 2] each, pairs of dimensions (i, i + rope_dim / 2), or (2 i, 2 i + 1) with
                   ``interleaved``; tokens behind the last position are not appended, and ``read_status`` tells

    What is returned is new, contiguous, rounded once, and zeros where a sequence has no token.  No two tokens of a call may be
    appended to the same place (sequences may share full pages).
    """
    _require(isinstance(cache, LatentCache), "the first argument must be a LatentCache")
    append, _, _, entries = _calls()
    if cache._writable:
        done = append(entries[0], cache._address, cache._index, cache._code, latents, rope_keys, table, lengths, counts, queries, rotation, interleaved)
        if done is not None:
            if done.__class__ is int:
                _lib.check(done)
            return done
    _check_rows(latents, "latents", cache.dtype, cache._index, (None, None, cache.latent_dim))
    B, T, _ = latents.shape
    _check_rows(rope_keys, "rope_keys", cache.dtype, cache._index, (B, T, cache.rope_dim))
    _require(cache._writable, "the rows of this cache lie on top of one another: it cannot be appended to")
    sequences = _sequences(cache, table, lengths, counts, B, T)
    rotated = q = None
    heads, q_strides = 0, (0, 0, 0)
    if queries is not None:
        _check_rows(queries, "queries", cache.dtype, cache._index, (B, T, None, cache.rope_dim))
        heads, q, q_strides = queries.shape[2], queries.data_ptr(), _strides(queries)
        rotated = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device)
    keys = torch.empty(B, T, cache.rope_dim, dtype=cache.dtype, device=cache.device)
    cos = sin = None
    positions = 0
    if rotation is not None:
        _require(isinstance(rotation, (tuple, list)) and len(rotation) == 2, "rotation must be (cos, sin)")
        cos, sin = rotation
        for t, name in ((cos, "cos"), (sin, "sin")):
            _require(isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.is_cuda and t.get_device() == cache._index,
                     f"{name} must be a float32 tensor on the cache's device")
            _require(t.dim() == 2 and t.shape[1] == cache.rope_dim // 2 and t.shape == cos.shape and t.shape[0] > 0 and t.is_contiguous()
                     and t.data_ptr() % 16 == 0, f"{name} must be contiguous, of shape [positions, rope_dim / 2], on a 16-byte boundary")
        positions = min(cos.shape[0], 0x7FFFFFFF)
        cos, sin = cos.data_ptr(), sin.data_ptr()
    _lib.check(_lib.load().fa_b200_latent_append(
        ctypes.byref(cache._handle), ctypes.byref(sequences), latents.data_ptr(), *_strides(latents), rope_keys.data_ptr(), *_strides(rope_keys), q, *q_strides, heads,
        keys.data_ptr(), None if rotated is None else rotated.data_ptr(), cos, sin, positions, _DTYPES[cache.dtype],
        _lib.CACHE_NEIGHBOURS if interleaved else 0, cache._index, _raw_stream(cache._index)))
    return keys, rotated


@lru_cache(maxsize=4096)
def _scratch_bytes(latent: int, heads: int, page: int, B: int, T: int, width: int, device: int) -> int:
    out = ctypes.c_uint64()
    _lib.check(_lib.load().fa_b200_latent_attention_scratch(latent, heads, page, B, T, width, device, ctypes.byref(out)))
    return out.value


def _check_scale(scale) -> float:
    _require(isinstance(scale, (int, float)) and 2.0 ** -126 <= scale <= 1e38, "scale must be a positive number, 2^-126 to 10^38")
    return float(scale)


def _check_out(out, like: torch.Tensor, shape, index: int) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _require(isinstance(out, torch.Tensor) and out.dtype == like.dtype and out.is_cuda and out.get_device() == index and tuple(out.shape) == tuple(shape)
             and out.is_contiguous() and out.data_ptr() % 16 == 0, f"out must be contiguous, of shape {list(shape)} and the queries' type")
    return out


def latent_attention(cache: LatentCache, q_latent: torch.Tensor, q_rope: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, scale: float,
                     counts: Optional[torch.Tensor] = None, causal: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of T queries a sequence over its latent vectors, [B, T, heads, latent_dim]: ``softmax(scale (q_latent . c + q_rope . r)) c``.

    ``q_latent`` [B, T, heads, latent_dim], the queries multiplied into the latent space;  ``q_rope`` [B, T, heads, rope_dim], rotated
    (``latent_append`` does that).  The queries are the last tokens of their sequences: query t stands at position ``lengths[b] - T + t``
    (``lengths[b] - counts[b] + t`` where ``counts`` says how many of the T a sequence has) and sees the rows up to its own; with
    ``causal=False`` all of its sequence.  ``scale`` is that of the heads' own keys, ``(nope + rope_dim) ** -0.5``.

    A query that sees nothing, or that its sequence does not have, gets zeros.  Rows that a query does not see do not reach it, whatever
    they hold.  Scores, maxima and sums are held in 32 bits; weights are rounded to the tensors' type for their product with the rows,
    and summed as rounded.
    """
    _require(isinstance(cache, LatentCache), "the first argument must be a LatentCache")
    _, attention, _, entries = _calls()
    y = attention(entries[1], entries[2], cache._address, cache._index, cache._code, q_latent, q_rope, table, lengths, scale, counts, causal, out)
    if y is not None:
        if y.__class__ is int:
            _lib.check(y)
        return y
    _check_rows(q_latent, "q_latent", cache.dtype, cache._index, (None, None, None, cache.latent_dim))
    B, T, heads, latent = q_latent.shape
    _check_rows(q_rope, "q_rope", cache.dtype, cache._index, (B, T, heads, cache.rope_dim))
    scale = _check_scale(scale)
    sequences = _sequences(cache, table, lengths, counts, B, T)
    out = _check_out(out, q_latent, (B, T, heads, latent), cache._index)
    scratch = torch.empty(_scratch_bytes(latent, heads, cache.page_size, B, T, table.shape[1], cache._index), dtype=torch.uint8, device=cache.device)
    _lib.check(_lib.load().fa_b200_latent_attention(
        ctypes.byref(cache._handle), ctypes.byref(sequences), q_latent.data_ptr(), *_strides(q_latent), q_rope.data_ptr(), *_strides(q_rope), heads, scale,
        _DTYPES[cache.dtype], 0 if causal else _lib.CACHE_ALL_KEYS, out.data_ptr(), scratch.data_ptr(), scratch.numel(), cache._index, _raw_stream(cache._index)))
    return out


def latent_prompt(q_nope: torch.Tensor, q_rope: torch.Tensor, expanded: torch.Tensor, rope_keys: torch.Tensor, *, scale: Optional[float] = None,
                  lengths: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, causal: bool = True,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of T queries a sequence with the keys and values of every head multiplied out of the latent vectors, [B, T, heads, nope_dim].

    ``q_nope``    [B, T, heads, nope_dim] (64 or 128);  ``q_rope`` [B, T, heads, rope_dim], rotated
    ``expanded``  [B, S, heads, 2 * nope_dim]: of each head its own part of the keys and behind it the values, ``latents @ W`` as it comes
    ``rope_keys`` [B, S, rope_dim], rotated (``latent_append`` returns those of its tokens): the rest of the keys, the same for all heads
    ``lengths``   int32 [B]: how many of the S tokens sequence b has (default: all);  ``counts`` int32 [B]: how many of the T queries (default: all)

    ``softmax(scale (q_nope . k + q_rope . r)) v``, with ``scale`` ``(nope_dim + rope_dim) ** -0.5`` unless given.  The queries are the last tokens of
    their sequences, as in ``latent_attention``, ``causal=False`` too.  A query that sees nothing, or that its sequence does not have, gets
    zeros.  Keys and values that a query does not see do not reach it, whatever they hold.  Scores, maxima and sums are held in 32 bits; weights
    are rounded to the tensors' type for their product with the values.  ``latent_status`` tells of lengths and counts outside, which are cut.
    """
    _, _, prompt, entries = _calls()
    y = prompt(entries[3], q_nope, q_rope, expanded, rope_keys, scale, lengths, counts, causal, out)
    if y is not None:
        if y.__class__ is int:
            _lib.check(y)
        return y
    _check_rows(q_nope, "q_nope", None, None, (None, None, None, None))
    B, T, heads, nope = q_nope.shape
    index, dtype = q_nope.get_device(), q_nope.dtype
    _require(nope in (64, 128), "nope_dim must be 64 or 128")
    _check_rows(q_rope, "q_rope", dtype, index, (B, T, heads, None))
    rope = q_rope.shape[3]
    _require(rope in ROPE_DIMS, "rope_dim must be 16, 32 or 64")
    _check_rows(expanded, "expanded", dtype, index, (B, None, heads, 2 * nope))
    S = expanded.shape[1]
    _check_rows(rope_keys, "rope_keys", dtype, index, (B, S, rope))
    for t, name in ((q_nope, "q_nope"), (q_rope, "q_rope"), (expanded, "expanded"), (rope_keys, "rope_keys")):
        _require(all(s > 0 or n == 1 for s, n in zip(t.stride(), t.shape)), f"the strides of {name} must be positive")
    for t, name in ((lengths, "lengths"), (counts, "counts")):
        if t is not None:
            _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.is_cuda and t.get_device() == index, f"{name} must be an int32 tensor on the queries' device")
            _require(tuple(t.shape) == (B,) and (B == 1 or t.stride(0) == 1), f"{name} must be contiguous, of shape [B]")
    scale = (nope + rope) ** -0.5 if scale is None else _check_scale(scale)
    out = _check_out(out, q_nope, (B, T, heads, nope), index)
    _lib.check(_lib.load().fa_b200_latent_prompt(
        q_nope.data_ptr(), *_strides(q_nope), q_rope.data_ptr(), *_strides(q_rope), expanded.data_ptr(), *_strides(expanded), rope_keys.data_ptr(), *_strides(rope_keys),
        None if lengths is None else lengths.data_ptr(), None if counts is None else counts.data_ptr(), B, T, S, heads, nope, rope, scale, _DTYPES[dtype],
        0 if causal else _lib.CACHE_ALL_KEYS, out.data_ptr(), index, _raw_stream(index)))
    return out


def latent_status(device: int = 0) -> Tuple[int, int]:
    """(first code, number of reports) of what ``latent_prompt``'s kernels found wrong on a device; clears it.  Synchronises.  The codes are those
    of ``cache.STATUS``."""
    out = (ctypes.c_uint32 * 2)()
    _lib.check(_lib.load().fa_b200_latent_status(device, out))
    return out[0], out[1]
