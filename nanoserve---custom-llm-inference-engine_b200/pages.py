"""Pages of a cache: copying, forking, compacting and freeing them.

The reference hands out fixed-size blocks of its key/value cache from a free
list (nanoserve/cache/block_allocator.py:14-47) and cannot share them between
requests.  Here:

* ``copy_pages`` copies pages of any number of pools (token ids, the keys and
  values of every layer) in one launch;
* ``gather_paged_history`` builds a step's CSR token histories out of pages;
* ``PageAllocator`` counts the users of each page on the host, so that
  requests can share the pages of a common prefix;
* ``PagedHistoryStore`` keeps the prior token ids of every request in pages,
  in place of ``HistoryStore``'s one region per request: a request
  reserves nothing ahead, can be forked, truncated and compacted, and caches
  that the same page table indexes move along.
"""
from __future__ import annotations

import contextlib
import heapq
from typing import Dict, Iterator, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _cabi, packing
from .history import StoreSampling
from .sampler import Sampler, _Op, _Staging, load_ops, upload_parts

_copy_pages = _Op("copy_pages")
_gather = _Op("paged_history_gather")

Pages = Union[Sequence[int], np.ndarray, torch.Tensor]


def _page_list(pages: Pages, name: str) -> torch.Tensor:
    if isinstance(pages, torch.Tensor):
        if pages.dtype == torch.int64 and pages.dim() == 1 and pages.is_cpu and pages.is_contiguous():
            return pages
        if pages.is_cuda:
            raise RuntimeError(f"{name} must be on the host: it is checked before anything is copied")
        if pages.dtype.is_floating_point or pages.dtype.is_complex or pages.dtype == torch.bool:
            raise ValueError(f"{name} must hold whole numbers")
        return pages.reshape(-1).to(torch.int64).contiguous()
    a = np.asarray(pages)
    if a.size and a.dtype.kind not in "iu":
        raise ValueError(f"{name} must hold whole numbers")
    return torch.from_numpy(np.ascontiguousarray(a.reshape(-1), dtype=np.int64))


def copy_pages(pools: Union[torch.Tensor, Sequence[torch.Tensor]], src: Pages, dst: Pages) -> None:
    """``pool[dst[j]] = pool[src[j]]`` for every pool and every ``j``.

    ``pools`` are CUDA tensors of any type on one device, with the page number
    as their first dimension, equally many pages, and each page contiguous
    (pages may be strided, as one half of a ``[pages, 2, ...]`` tensor is; pools must not
    overlap one another, but for one that is named twice).
    ``src`` and ``dst`` are lists, arrays or CPU tensors of page numbers.  A page
    may be copied to several places; ``ValueError`` is raised, and nothing
    copied, where a page does not exist, is a destination twice, or is both a
    source and a destination.  One launch per 64 pools on the current stream of
    the pools' device (lists of more than 3500 pages are uploaded first, or, in a
    stream capture, take a launch per 3500); the page numbers are taken during
    the call, so a graph that captures it replays the same copies."""
    s, d = _page_list(src, "src"), _page_list(dst, "dst")
    _copy_pages([pools] if isinstance(pools, torch.Tensor) else pools, s, d)


def gather_paged_history(
    pool: torch.Tensor,
    pages: torch.Tensor,
    page_offsets: torch.Tensor,
    history_offsets: torch.Tensor,
    *,
    out: torch.Tensor,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """A step's CSR history ids out of a paged pool: for row ``r`` and ``j < history_offsets[r+1] -
    history_offsets[r]``, ``out[history_offsets[r] + j]`` is token ``j % page_size`` of page
    ``pages[page_offsets[r] + j // page_size]``.

    Device tensors: ``pool`` int32 ``[num_pages, page_size]``, ``pages`` int32 (all rows' page tables,
    one after the other), ``page_offsets`` and ``history_offsets`` int64 ``[S+1]``, ``out`` int32 with room
    for ``history_offsets[S]`` ids; ids behind them are left as they were.  Offsets must not fall (that sets
    the status, and rows are left out).  Where a table is too short or a
    page does not exist the id becomes -1 (which the sampler reports) and ``NS_STATUS_BAD_POOL_RANGE`` is
    set in ``status`` (int32 ``[1]``).  One launch on the current stream of ``pool.device``."""
    _gather(pool, pages, page_offsets, history_offsets, out, status)
    return out


class PageAllocator:
    """Free list of ``num_pages`` pages with a count of each page's users (host
    bookkeeping only).  The lowest free page is handed out first."""

    def __init__(self, num_pages: int):
        if num_pages < 0:
            raise ValueError("num_pages must be >= 0")
        self.num_pages = int(num_pages)
        self._users = np.zeros(self.num_pages, dtype=np.int32)
        self._free: List[int] = list(range(self.num_pages))  # a heap

    def alloc(self, n: int) -> List[int]:
        """``n`` free pages, one user each; MemoryError (and no page taken) if there are fewer."""
        if n < 0:
            raise ValueError("n must be >= 0")
        if n > len(self._free):
            raise MemoryError(f"page pool full: {n} pages asked for, {len(self._free)} of {self.num_pages} free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        self._users[got] = 1
        return got

    def users(self, page: int) -> int:
        return int(self._users[page])

    def share(self, pages: Sequence[int]) -> None:
        """One more user of each of these pages."""
        for p in pages:
            if not 0 <= p < self.num_pages or self._users[p] <= 0:
                raise ValueError(f"page {p} is not in use")
        for p in pages:
            self._users[p] += 1

    def free(self, pages: Sequence[int]) -> None:
        """One user fewer of each of these pages; a page without users is free again."""
        gone: Dict[int, int] = {}
        for p in pages:
            gone[p] = gone.get(p, 0) + 1
        for p, k in gone.items():
            if not 0 <= p < self.num_pages or self._users[p] < k:
                raise ValueError(f"page {p} is freed more often than it was taken")
        for p, k in gone.items():
            self._users[p] -= k
            if self._users[p] == 0:
                heapq.heappush(self._free, p)

    def free_total(self) -> int:
        return len(self._free)

    def live_total(self) -> int:
        return self.num_pages - len(self._free)

    def plan_compact(self) -> Tuple[np.ndarray, np.ndarray]:
        """The fewest moves (src, dst) after which the live pages are ``0 .. live_total() - 1``."""
        live = self.live_total()
        used = self._users > 0
        return live + np.flatnonzero(used[live:]), np.flatnonzero(~used[:live])

    def move(self, src: np.ndarray, dst: np.ndarray) -> None:
        """Take over the moves of ``plan_compact``."""
        self._users[dst] = self._users[src]
        self._users[src] = 0
        self._free = np.flatnonzero(self._users == 0).tolist()  # ascending: a heap


class _Request:
    __slots__ = ("pages", "length", "prompt")

    def __init__(self, pages: List[int], length: int, prompt: int):
        self.pages, self.length, self.prompt = pages, length, prompt


class PagedHistoryStore(StoreSampling):
    """Prior-token histories in pages of one int32 device pool, shared between
    forks of a request.

    ``caches`` are further pools that the same pages index (``[num_pages, ...]``, as
    the keys and values of an engine's layers): forking, truncating and
    compacting copies their pages along; ``pages(handle)`` is the request's page
    table.  A page with several users is never written: the page that a request's next
    token goes to is its own.

    Calls are enqueued on the current stream of the store's device; use one
    stream, or order them, as for any tensor."""

    def __init__(self, device, num_pages: int, vocab: int, page_size: int = 16,
                 caches: Sequence[torch.Tensor] = ()):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedHistoryStore keeps its pool on a CUDA device (no CPU fallback)")
        if page_size <= 0:
            raise ValueError("page_size must be positive")
        load_ops()
        self.vocab, self.num_pages, self.page_size = int(vocab), int(num_pages), int(page_size)
        self.caches = list(caches)
        for c in self.caches:
            if c.dim() == 0 or c.shape[0] != self.num_pages:
                raise ValueError(f"a cache of shape {tuple(c.shape)} does not have {self.num_pages} pages")
        self.pool = torch.zeros(self.num_pages, self.page_size, dtype=torch.int32, device=self.device)
        self.device = self.pool.device
        copy_pages([self.pool, *self.caches], [], [])  # refuses caches that cannot be copied with the pool
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._alloc = PageAllocator(self.num_pages)
        self._requests: Dict[int, _Request] = {}
        self._next = 0
        self._staging = _Staging()
        self._append_staging = _Staging()
        self._ids: Optional[torch.Tensor] = None

    # -- requests -----------------------------------------------------------
    def _needed(self, length: int) -> int:
        return -(-length // self.page_size)

    @contextlib.contextmanager
    def _taken(self, n: int) -> Iterator[List[int]]:
        """``n`` pages, given back if the copies that fill them fail; the store's device is current."""
        pages = self._alloc.alloc(n)
        try:
            with torch.cuda.device(self.device):
                yield pages
        except BaseException:
            self._alloc.free(pages)
            raise

    def _new(self, request: _Request) -> int:
        h = self._next
        self._next += 1
        self._requests[h] = request
        return h

    def add(self, prompt_ids: Sequence[int], max_new_tokens: int = 0) -> int:
        """A new request with these ids; pages for ``max_new_tokens`` more are taken now,
        further ones as they are needed."""
        ids = np.asarray(prompt_ids, dtype=np.int64).reshape(-1)
        if ids.size and (int(ids.min()) < 0 or int(ids.max()) >= self.vocab):
            bad = int(ids.min()) if int(ids.min()) < 0 else int(ids.max())
            raise IndexError(f"history token id {bad} is out of range for vocab size {self.vocab}")
        if max_new_tokens < 0:
            raise ValueError("max_new_tokens must be >= 0")
        n = self._needed(ids.size)
        with self._taken(self._needed(ids.size + max_new_tokens)) as pages:
            if n:
                rows = np.zeros((n, self.page_size), dtype=np.int32)
                rows.reshape(-1)[: ids.size] = ids
                at = torch.tensor(pages[:n], dtype=torch.int64).pin_memory().to(self.device, non_blocking=True)
                self.pool[at] = torch.from_numpy(rows).pin_memory().to(self.device, non_blocking=True)
        return self._new(_Request(pages, int(ids.size), int(ids.size)))

    def fork(self, handle: int, n: int = 1) -> List[int]:
        """``n`` new requests with ``handle``'s ids so far: they share its full pages, and its
        last page, if it is not full, is copied for each (one launch)."""
        if n < 0:
            raise ValueError("n must be >= 0")
        r = self._requests[handle]
        full, rest = divmod(r.length, self.page_size)
        with self._taken(n if rest else 0) as own:
            if own:
                copy_pages([self.pool, *self.caches], [r.pages[full]] * n, own)
        out = []
        for i in range(n):
            self._alloc.share(r.pages[:full])
            out.append(self._new(_Request(r.pages[:full] + own[i : i + 1], r.length, r.prompt)))
        return out

    def reserve(self, handle: int, tokens: int) -> None:
        """Take the pages for ``tokens`` more ids now (for caches that are written ahead of ``append``)."""
        if tokens < 0:
            raise ValueError("tokens must be >= 0")
        r = self._requests[handle]
        r.pages += self._alloc.alloc(max(0, self._needed(r.length + tokens) - len(r.pages)))

    def truncate(self, handle: int, length: int) -> None:
        """Keep the first ``length`` ids (as after rejected speculative tokens); the pages behind
        them are freed.  A last page that forks share becomes the request's own copy."""
        r = self._requests[handle]
        if not 0 <= length <= r.length:
            raise ValueError(f"length must be between 0 and {r.length}, got {length}")
        keep = self._needed(length)
        kept, gone = r.pages[:keep], r.pages[keep:]
        if length % self.page_size and self._alloc.users(kept[-1]) > 1:
            mine = [p for p in gone if self._alloc.users(p) == 1][:1]
            with self._taken(1 - len(mine)) as new:
                own = (mine + new)[0]
                copy_pages([self.pool, *self.caches], [kept[-1]], [own])
            gone = [p for p in gone if p != own] + [kept[-1]]
            kept[-1] = own
        self._alloc.free(gone)
        r.pages, r.length, r.prompt = kept, int(length), min(r.prompt, int(length))

    def release(self, handle: int) -> None:
        self._alloc.free(self._requests.pop(handle).pages)

    def compact(self) -> int:
        """Move the live pages to the front of the pool and of the caches; returns how many moved.  Page tables taken before are stale."""
        src, dst = self._alloc.plan_compact()
        if src.size:
            with torch.cuda.device(self.device):
                copy_pages([self.pool, *self.caches], src, dst)
            to = np.arange(self.num_pages)
            to[src] = dst
            for r in self._requests.values():
                r.pages = to[r.pages].tolist() if r.pages else []
            self._alloc.move(src, dst)
        return int(src.size)

    def length(self, handle: int) -> int:
        return self._requests[handle].length

    def prompt_length(self, handle: int) -> int:
        return self._requests[handle].prompt

    def pages(self, handle: int) -> List[int]:
        """The request's page table: page ``i`` holds ids ``i * page_size`` and on."""
        return list(self._requests[handle].pages)

    def free_pages(self) -> int:
        return self._alloc.free_total()

    def tokens(self, handle: int) -> List[int]:
        """The request's ids as a list (synchronises; for tests and debugging)."""
        r = self._requests[handle]
        at = torch.tensor(r.pages[: self._needed(r.length)], dtype=torch.int64, device=self.device)
        return self.pool[at].reshape(-1)[: r.length].tolist()

    # -- one step -----------------------------------------------------------
    def _history_parts(self, handles: Sequence[int], lens: np.ndarray) -> List[np.ndarray]:
        need = -(-lens // self.page_size)
        page_offsets = np.zeros(len(handles) + 1, dtype=np.int64)
        np.cumsum(need, out=page_offsets[1:])
        pages = np.zeros(int(page_offsets[-1]), dtype=np.int32)
        for i in np.flatnonzero(need):
            pages[page_offsets[i] : page_offsets[i + 1]] = self._requests[handles[i]].pages[: need[i]]
        return [page_offsets, pages]

    def _history_ids(self, parts: Sequence[torch.Tensor], offsets: torch.Tensor, ids: torch.Tensor) -> None:
        gather_paged_history(self.pool, parts[1], parts[0], offsets, out=ids, status=self.status)

    def _grow(self, handles: Sequence[int]) -> None:
        """A page for the next token of each of these requests (all of them, or MemoryError and none)."""
        if len(set(handles)) != len(handles):
            raise ValueError("a request appears twice")
        grow = [r for r in (self._requests[h] for h in handles) if r.length == len(r.pages) * self.page_size]
        for r, p in zip(grow, self._alloc.alloc(len(grow))):
            r.pages.append(p)

    def sample(self, sampler: Sampler, logits: torch.Tensor, sampling_params_list: Sequence, handles: Sequence[int],
               *, append: bool = True, **kw):
        if append:
            self._grow(handles)  # a full pool is found out before anything is sampled
        return super().sample(sampler, logits, sampling_params_list, handles, append=append, **kw)

    sample.__doc__ = StoreSampling.sample.__doc__

    def append(self, handles: Sequence[int], tokens: torch.Tensor) -> None:
        """Append ``tokens[i]`` (device int64 or int32 [S]) to request ``handles[i]``."""
        S = len(handles)
        if tokens.numel() != S or tokens.device != self.device:
            raise ValueError("tokens must be a device tensor with one id per handle")
        if tokens.dtype not in (torch.int64, torch.int32):
            raise ValueError("tokens must be int64 or int32")
        self._grow(handles)
        reqs = [self._requests[h] for h in handles]
        dst = np.fromiter((r.pages[r.length // self.page_size] * self.page_size + r.length % self.page_size
                           for r in reqs), dtype=np.int64, count=S)
        with torch.cuda.device(self.device):
            (dev,) = upload_parts(self._append_staging, [dst], self.device)
            tokens = tokens.contiguous()
            _cabi.ns_history_append(self.pool.data_ptr(), self.num_pages * self.page_size, dev.data_ptr(),
                                    tokens.data_ptr(),
                                    _cabi.NS_OUT_I32 if tokens.dtype == torch.int32 else _cabi.NS_OUT_I64, S,
                                    self.status.data_ptr(), torch.cuda.current_stream(self.device).cuda_stream)
        for r in reqs:
            r.length += 1
