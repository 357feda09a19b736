"""The pages of a cache: who holds them, forks that share them, pages of one's own before writing, moving them to the front.

A ``PagePool`` counts for each page of a program's caches (all layers' alike) how many entries of the table hold it.  The table is the one
that the caches' calls take, int32 [B, W] on the device with the page of the i-th block of sequence b in ``table[b, i]``; -1 is no page.

  pool = page_pool_create(n_pages)
  table, lengths = torch.full((B, W), -1, ...), torch.zeros(B, ...)
  granted, sources, targets = pages_reserve(pool, table, lengths, counts, page_size)     # pages for counts[b] more tokens
  cache_copy(caches, sources, targets)                                                   # what shared pages held
  cache_append(cache, k, v, table, lengths, counts=granted)                              # for every layer
  lengths += granted
  pages_fork(pool, table, lengths, parents)                                              # beams; -1 lets a sequence go
  pool, table, sources, targets = pages_compact(pool, table)                             # then cache_copy, and on with these

Nothing is read on the host; all calls are asynchronous on the current stream and can be captured.  The program orders calls on one pool and
table by streams.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Tuple, Union

import torch

from . import _lib
from .api import _load_native, _raw_stream
from .cache import PAGE_SIZES, KVCache
from .latent import LatentCache

# What the first status word of a pool stands for (fa_pages.cuh).
STATUS = {0: "nothing", 1: "a table entry that is neither a page nor -1", 2: "a length, count or parent outside", 3: "no page was free",
          4: "counts that do not fit the table"}


_native = None   # the extension module's calls, and the library's entries that they go to


def _require(cond: bool, what: str) -> None:
    if not cond:
        raise RuntimeError(f"pages: {what}")


def _calls():
    """(fork, reserve, compact, copy, entries): as in cache.py, None is the answer to what goes through the checks and ctypes below, an int the
    status of a launch that failed."""
    global _native
    if _native is None:
        lib = _lib.load()   # raises when the CUDA library is missing: no fallback
        _native = tuple(_load_native(name) for name in ("_pages_fork_through", "_pages_reserve_through", "_pages_compact_through", "_cache_copy_through")) + (lib.pages_entries,)
    return _native


def _done(answer) -> bool:
    if answer.__class__ is int:
        _lib.check(answer)
    return answer is not None


class PagePool:
    """How many table entries hold each page: ``refs``, int32 [n_pages], contiguous; 0 is a free page."""

    def __init__(self, refs: torch.Tensor):
        _require(isinstance(refs, torch.Tensor) and refs.dtype == torch.int32, "refs must be an int32 tensor")
        _require(refs.is_cuda, "refs must be a CUDA tensor")
        _require(refs.dim() == 1 and 0 < refs.shape[0] < 1 << 30 and refs.is_contiguous(), "refs must be contiguous, of shape [n_pages]")
        self._set(refs, refs.shape[0], refs.device, refs.get_device(), torch.zeros(4, dtype=torch.int32, device=refs.device))

    def _set(self, refs, n_pages, device, index, status) -> "PagePool":
        self.refs, self.n_pages, self.device, self._index, self._status = refs, n_pages, device, index, status
        self._handle = _lib.Pages(refs.data_ptr(), status.data_ptr(), n_pages)
        self._address = ctypes.addressof(self._handle)
        return self

    def _with(self, refs: torch.Tensor) -> "PagePool":
        """A pool of other counts of the same pages, which reports where this one does; otherwise calls on the two have nothing in common."""
        return PagePool.__new__(PagePool)._set(refs, self.n_pages, self.device, self._index, self._status)

    def read_status(self) -> Tuple[int, int]:
        """(first code, number of reports) of what the kernels found wrong; clears it.  Synchronises.  ``STATUS`` says what the codes mean."""
        code, reports = self._status[:2].tolist()
        if code or reports:
            self._status[:2].zero_()
        return code, reports


def page_pool_create(n_pages: int, device="cuda") -> PagePool:
    """A pool whose pages are all free."""
    _require(0 < n_pages < 1 << 30, "n_pages must be positive and below 2^30")
    return PagePool(torch.zeros(n_pages, dtype=torch.int32, device=device))


def _check_ints(t, name: str, pool: PagePool, shape, writable: bool = False) -> None:
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32, f"{name} must be an int32 tensor")
    _require(t.is_cuda and t.get_device() == pool._index, f"{name} must be on the pool's device")
    _require(t.dim() == len(shape) and all(n is None or t.shape[i] == n for i, n in enumerate(shape)) and 0 not in t.shape,
             f"{name} must have shape {['B', 'W'][:len(shape)]}" + ("" if shape[0] is None else f", B {shape[0]}"))
    _require(t.shape[-1] == 1 or t.stride(-1) == 1, f"the last axis of {name} must be contiguous")
    if writable and t.dim() == 2:
        _require(t.shape[0] == 1 or abs(t.stride(0)) >= t.shape[1], f"the rows of {name} lie on top of one another: it cannot be written to")


def pages_fork(pool: PagePool, table: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor) -> None:
    """Every sequence goes on as its parent: row b of ``table`` becomes what row ``parents[b]`` was, ``lengths[b]`` what its length was, all at
    once and in place; a parent of -1 lets the sequence go (its row becomes -1, its length 0).

    ``parents`` int32 [B]: b itself where nothing changes.  Pages are shared, not copied: ``pages_reserve`` gives those that will be
    written to a page of their own.  At most 57344 sequences.
    """
    _require(isinstance(pool, PagePool), "the first argument must be a PagePool")
    fork, _, _, _, entries = _calls()
    done = fork(entries[0], pool._address, pool._index, table, lengths, parents)
    if _done(done):
        return
    _check_ints(table, "table", pool, (None, None), True)
    B, W = table.shape
    _check_ints(lengths, "lengths", pool, (B,))
    _check_ints(parents, "parents", pool, (B,))
    _require(B <= 57344, "at most 57344 sequences")
    _lib.check(_lib.load().fa_b200_pages_fork(ctypes.byref(pool._handle), table.data_ptr(), table.stride(0), W, B, lengths.data_ptr(), parents.data_ptr(), pool._index,
                                              _raw_stream(pool._index)))


def pages_reserve(pool: PagePool, table: torch.Tensor, lengths: torch.Tensor, counts: Union[torch.Tensor, int],
                  page_size: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Give every sequence the blocks that ``lengths[b] + counts[b]`` tokens need, and no more; (granted, sources, targets), int32 [B] each.

    ``counts`` int32 [B], or a number for all: how many tokens will be appended.  Blocks behind them are let go of (drafted tokens that were
    taken back by lowering ``lengths``; with ``counts`` 0 and a length of 0 a whole sequence).  Blocks that the new tokens go to
    and that have no page get one; so do those whose page others hold too, unless all that hold it are about to write to it: then the
    sequence with the most tokens on it keeps it, the lowest of several.  New pages are the lowest free ones in order of sequences and
    blocks.  Where such a block holds tokens already, sources[b] is the page that it was on and targets[b] the new one (-1 elsewhere):
    ``cache_copy`` has to come before the append.

    ``granted[b]`` is counts[b], or fewer where pages ran out (or the table has no room): the ``counts`` of ``cache_append``.  A sequence that finds
    no page in place of a shared one stays on it with the tokens it has; whoever keeps the page goes on behind all of them.  (The scales of an
    8-bit cache are the page's: what goes on there may enlarge them, as tokens that were taken back may have.)
    """
    _require(isinstance(pool, PagePool), "the first argument must be a PagePool")
    _, reserve, _, _, entries = _calls()
    done = reserve(entries[1], pool._address, pool._index, table, lengths, counts, page_size)
    if _done(done):
        return done
    _check_ints(table, "table", pool, (None, None), True)
    B, W = table.shape
    _check_ints(lengths, "lengths", pool, (B,))
    _require(isinstance(page_size, int) and page_size in PAGE_SIZES, "page_size must be 16, 32, 64 or 128")
    given = isinstance(counts, torch.Tensor)
    if given:
        _check_ints(counts, "counts", pool, (B,))
    else:
        _require(isinstance(counts, int) and 0 <= counts <= 0x7FFFFFFF, "counts must be an int32 tensor or a number that is not negative")
    granted, sources, targets = torch.empty(3, B, dtype=torch.int32, device=pool.device).unbind(0)
    scratch = torch.empty(pool.n_pages, dtype=torch.int32, device=pool.device)
    _lib.check(_lib.load().fa_b200_pages_reserve(
        ctypes.byref(pool._handle), table.data_ptr(), table.stride(0), W, B, lengths.data_ptr(), counts.data_ptr() if given else None, 0 if given else counts, page_size,
        granted.data_ptr(), sources.data_ptr(), targets.data_ptr(), scratch.data_ptr(), 4 * scratch.numel(), pool._index, _raw_stream(pool._index)))
    return granted, sources, targets


def pages_compact(pool: PagePool, table: torch.Tensor) -> Tuple[PagePool, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the pages that are held to the front of the caches: (pool, table, sources, targets) as they are afterwards.

    With n pages held, the k-th of those from page n on goes to the k-th free one in front of it.  ``sources`` and ``targets``, int32 [n_pages],
    are the moves, -1 behind the last: after ``cache_copy(caches, sources, targets)`` the program goes on with the new pool and table.  The
    old ones are left as they are.  Beyond 100000 pages time grows with their square: 0.2 ms for a million, 2 for 4 million.
    """
    _require(isinstance(pool, PagePool), "the first argument must be a PagePool")
    _, _, compact, _, entries = _calls()
    done = compact(entries[2], pool._address, pool._index, table)
    if _done(done):
        return (pool._with(done[0]),) + done[1:]
    _check_ints(table, "table", pool, (None, None))
    B, W = table.shape
    refs, sources, targets = torch.empty(3, pool.n_pages, dtype=torch.int32, device=pool.device).unbind(0)
    new = torch.empty(B, W, dtype=torch.int32, device=pool.device)
    scratch = torch.empty(pool.n_pages + 2, dtype=torch.int32, device=pool.device)
    _lib.check(_lib.load().fa_b200_pages_compact(
        ctypes.byref(pool._handle), table.data_ptr(), table.stride(0), W, B, refs.data_ptr(), new.data_ptr(), sources.data_ptr(), targets.data_ptr(),
        scratch.data_ptr(), 4 * scratch.numel(), pool._index, _raw_stream(pool._index)))
    return pool._with(refs), new, sources, targets


def _areas(cache):
    """(address, how many, the array itself): the arrays of a cache's pages as the library copies them; made once for each cache."""
    if cache._copy_areas is None:
        if isinstance(cache, KVCache):
            n, heads, page, H = cache.k.shape
            areas = [_lib.CopyArea(t.data_ptr(), *t.stride()[:3], heads, page, H) for t in (cache.k, cache.v)]
            # (a row a head, because scales may start on any 4-byte boundary; the library takes them in one where that can be)
            areas += [_lib.CopyArea(t.data_ptr(), 4 * heads, 0, 4, 1, heads, 4) for t in (cache.k_scale, cache.v_scale)]
            areas.append(_lib.CopyArea(cache.bounds.data_ptr(), 2 * H * heads, 0, 0, 1, 1, 2 * H * heads))
        else:
            n, page, width = cache.data.shape
            areas = [_lib.CopyArea(cache.data.data_ptr(), 2 * cache.data.stride(0), 2 * cache.data.stride(1), 0, page, 1, 2 * width)]
        array = (_lib.CopyArea * len(areas))(*areas)
        cache._copy_areas = (ctypes.addressof(array), len(areas), array)
    return cache._copy_areas


def cache_copy(caches, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Copy the contents of page ``sources[i]`` to page ``targets[i]``, in one cache or in every one of a list (the layers').

    ``sources``, ``targets`` int32 [n] on the caches' device; pairs with -1 are passed over.  No page may be a target twice, or a target and
    a source.  The caches have as many pages each; a page outside is reported in the first one's ``read_status``.
    """
    if caches.__class__ not in (list, tuple):
        caches = (caches,)
    _require(len(caches) > 0 and isinstance(caches[0], (KVCache, LatentCache)), "the first argument must be a KVCache, a LatentCache or a list of them")
    first = caches[0]
    areas = []
    for c in caches:
        _require(isinstance(c, (KVCache, LatentCache)), "the first argument must be a KVCache, a LatentCache or a list of them")
        _require(c.n_pages == first.n_pages and c._index == first._index, "the caches must have as many pages, on one device")
        _require(c._writable, "the pages of a cache lie on top of one another: it cannot be copied to")
        areas.append(c._copy_areas or _areas(c))
    areas, status = tuple(areas), first._status.data_ptr()
    _, _, _, copy, entries = _calls()
    if _done(copy(entries[3], areas, first.n_pages, status, first._index, sources, targets)):
        return
    for t, name in ((sources, "sources"), (targets, "targets")):
        _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.is_cuda and t.get_device() == first._index,
                 f"{name} must be an int32 tensor on the caches' device")
        _require(t.dim() == 1 and t.shape[0] > 0 and (t.shape[0] == 1 or t.stride(0) == 1), f"{name} must be contiguous, of shape [n]")
    _require(sources.shape == targets.shape, "targets must have the shape of sources")
    both = [a for _, _, array in areas for a in array]
    _lib.check(_lib.load().fa_b200_cache_copy((_lib.CopyArea * len(both))(*both), len(both), first.n_pages, sources.data_ptr(), targets.data_ptr(), sources.shape[0],
                                              status, first._index, _raw_stream(first._index)))
