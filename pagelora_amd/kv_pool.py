"""Paged KV pool, page allocator and per-request spans.

Layout of the pool (``model/kvcache/paged_kv_store.py:559-570``): one dense
tensor ``[num_layers, capacity_pages, 2, page_size, num_kv_heads, head_dim]``;
``pool[l]`` is the NHD layer view the decode kernels read, with K at index
0 and V at index 1 of dim 2 (``layer_runner.py:411-412``).

Size the pool for the whole workload up front (288 GB of HBM makes that
the normal case): its data pointer then stays fixed and a captured decode
graph replays for the life of the engine.  When it does run out, it grows
as the reference's does (``paged_kv_store.py:304-330, 543-579``): a new
tensor of ``max(16, 2 x capacity, required)`` pages, or exactly
``max_pages`` when capped, with the old pages copied in place, so every
page id stays valid.  The move changes the pool's data pointer, which is
part of every decode graph key, so the next step recaptures once.

Requests own page spans (``KVBlockSpan``); rows may share prefix pages
(``paged_kvcache_manager.py:324-333``), which are read-only to decode.

Requests can also be forked, cut back and packed together.  A fork shares the
full pages of its own with its origin, counted, and gets a copy of the page
they would both write to; a page goes back to the free list with its last
holder.  The copies run on the device, in all layers at once.
"""

from __future__ import annotations

import math
from array import array
from dataclasses import dataclass, field
from typing import Sequence

import numpy as np
import torch

from . import _lib
from .page_table import KVBlockSpan, pack_rows


def kv_copy_pages(cache: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
    """Make page ``dst[i]`` a copy of page ``src[i]`` in every layer (``pl_kv_copy_pages``).

    ``cache``: the pool [layers, P, 2, page, Hkv, D], or one layer of it, its
    pages contiguous.  Page ids are host integers.  A source may be listed more
    than once; a page that is written must not be written twice nor be a
    source.  Enqueued on the current stream; the lists are read at once.
    """

    shape, strides = cache.shape, cache.stride()
    if len(shape) == 5:
        shape, strides = (1, *shape), (0, *strides)
    if len(shape) != 6 or shape[2] != 2:
        raise ValueError(f"cache must be [layers, P, 2, page, Hkv, D] or a layer of it, got {tuple(cache.shape)}")
    try:
        src, dst = array("i", src), array("i", dst)
    except (TypeError, OverflowError):
        raise ValueError("page ids must be integers of 32 bits") from None
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} source pages but {len(dst)} destination pages")
    if not src:
        return
    device = cache.get_device()
    if device < 0:
        raise RuntimeError("kv_copy_pages needs a cache on a ROCm device")
    page = math.prod(shape[2:])
    # (the stride of a dim of one entry says nothing)
    if any(n > 1 and a != b for n, a, b in zip(shape[2:], strides[2:], (page // 2, shape[4] * shape[5], shape[5], 1))):
        raise ValueError("the pages of the KV cache must be contiguous")
    with _lib.on_device(device):
        _lib.check(_lib.load().pl_kv_copy_pages(
            cache.data_ptr(), strides[0], strides[1], page, shape[0], shape[1], src.buffer_info()[0],
            dst.buffer_info()[0], len(src), _lib.dtype_code(cache.dtype), _lib.raw_stream(device)),
            "pl_kv_copy_pages")


class PageAllocator:
    """Free-list page allocator (paged_kv_allocator.py:22-73 semantics:
    allocate n pages or fail atomically, free returns pages to the list).

    Page 0 is never handed out: it is the scratch slot that graph warm-up
    runs append their (discarded) K/V into.  ``grow(required_pages)``, when
    given, is called when the free list runs short; it returns the new
    capacity, whose pages join the free list (lowest ids handed out first).

    An allocated page has one holder; :meth:`share` adds one, :meth:`free`
    takes one away, and the last one's free returns the page to the list.
    """

    def __init__(self, capacity: int, grow=None) -> None:
        self.capacity = int(capacity)
        self._free = list(range(self.capacity - 1, 0, -1))
        self._grow = grow
        self._more: dict[int, int] = {}  # holders of a page beyond the first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def allocate(self, n: int) -> list[int]:
        if n > len(self._free):
            if self._grow is None:
                raise RuntimeError(f"paged KV pool exhausted: need {n} pages, {len(self._free)} free")
            new_cap = int(self._grow(self.capacity + n - len(self._free)))
            self._free = list(range(new_cap - 1, self.capacity - 1, -1)) + self._free
            self.capacity = new_cap
        out = [self._free.pop() for _ in range(n)]
        return out

    def share(self, pages) -> None:
        """One holder more for each of these allocated pages."""
        for p in pages:
            self._more[int(p)] = self._more.get(int(p), 0) + 1

    def holders(self, page: int) -> int:
        """How many hold an allocated page."""
        return 1 + self._more.get(int(page), 0)

    def free(self, pages) -> None:
        for p in map(int, pages):
            more = self._more.get(p, 0)
            if more == 0:
                self._free.append(p)
            elif more == 1:
                del self._more[p]
            else:
                self._more[p] = more - 1

    def move(self, moved: dict[int, int]) -> None:
        """Allocated pages ``moved`` (page -> free page) take those ids; the
        free list hands out the lowest ids first again."""
        free = set(self._free) - set(moved.values()) | set(moved)
        self._free = sorted(free, reverse=True)
        self._more = {moved.get(p, p): n for p, n in self._more.items()}


@dataclass
class Request:
    """One sequence's pages: shared prefix pages (read-only) + own pages."""

    prefix_pages: list[int] = field(default_factory=list)
    prefix_len: int = 0          # tokens held by the prefix pages (a multiple of page_size)
    own_pages: list[int] = field(default_factory=list)
    length: int = 0              # total tokens (prefix + own)

    def pages(self) -> list[int]:
        return self.prefix_pages + self.own_pages

    def spans(self, page_size: int) -> list[KVBlockSpan]:
        out = []
        remaining = self.length
        for p in self.pages():
            n = min(page_size, remaining)
            if n <= 0:
                break
            out.append(KVBlockSpan(p, 0, n))
            remaining -= n
        return out

    def slot(self, position: int, page_size: int) -> tuple[int, int]:
        """(page id, offset) that holds logical token ``position``."""
        return self.pages()[position // page_size], position % page_size


class PagedKVPool:
    """Paged KV pool for all layers plus its allocator.

    ``max_pages``: 0 grows without bound (the reference's default), > 0
    grows straight to that many pages and no further, None never grows (an
    exhausted pool raises RuntimeError).
    """

    def __init__(
        self,
        *,
        num_layers: int,
        capacity_pages: int,
        page_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device | str,
        max_pages: int | None = 0,
    ) -> None:
        if max_pages is not None and max_pages > 0 and max_pages < capacity_pages:
            raise ValueError(f"max_pages {max_pages} < capacity_pages {capacity_pages}")
        self.num_layers = num_layers
        self.page_size = page_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.cache = torch.empty(
            (num_layers, capacity_pages, 2, page_size, num_kv_heads, head_dim), dtype=dtype, device=device
        )
        self.max_pages = max_pages
        self.version = 0      # bumped whenever the pool tensor moves
        self.grow_count = 0
        self.allocator = PageAllocator(capacity_pages, grow=None if max_pages is None else self._grow)

    def _grow(self, required_pages: int) -> int:
        """Move the pool to a larger tensor, copying every page (ids unchanged)
        (paged_kv_store.py:543-579: max(16, 2 x capacity, required), or
        exactly max_pages when capped).  Stream-ordered: work queued earlier
        on the current stream finishes with the old tensor first."""
        cap = self.capacity_pages
        if self.max_pages:
            if required_pages > self.max_pages:
                raise RuntimeError(f"paged KV pool capacity exceeded: {required_pages} pages > max_pages "
                                   f"{self.max_pages}")
            new_cap = self.max_pages
        else:
            new_cap = max(16, 2 * cap, required_pages)
        old = self.cache
        new = torch.empty((old.shape[0], new_cap) + tuple(old.shape[2:]), dtype=old.dtype, device=old.device)
        new[:, :cap].copy_(old)
        self.cache = new
        self.version += 1
        self.grow_count += 1
        return new_cap

    @property
    def capacity_pages(self) -> int:
        return self.cache.shape[1]

    def layer_cache(self, layer: int) -> torch.Tensor:
        return self.cache[layer]

    def reserve(self, request: Request, new_tokens: int) -> None:
        """Grow the request by ``new_tokens`` tokens, allocating pages as needed."""
        need = -(-(request.length + new_tokens - request.prefix_len) // self.page_size) - len(request.own_pages)
        if need > 0:
            request.own_pages += self.allocator.allocate(need)
        request.length += new_tokens

    def release(self, request: Request) -> None:
        self.allocator.free(request.own_pages)
        request.own_pages = []

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Page ``dst[i]`` becomes a copy of page ``src[i]`` in every layer (:func:`kv_copy_pages`)."""
        kv_copy_pages(self.cache, src, dst)

    def fork(self, requests: Sequence[Request]) -> list[Request]:
        """A continuation of its own for each request (listed n times: n of
        them), with the same tokens so far.  Full pages are shared, a partial
        last page is copied: one launch for all of them, in stream order."""
        partial = [r.length % self.page_size > 0 and r.length > r.prefix_len for r in requests]
        full = [max(0, r.length - r.prefix_len) // self.page_size for r in requests]
        src = [r.own_pages[n] for r, n, cut in zip(requests, full, partial) if cut]
        dst = self.allocator.allocate(len(src))
        try:
            self.copy_pages(src, dst)
        except Exception:
            self.allocator.free(dst)
            raise
        copies = iter(dst)
        forks = []
        for r, n, cut in zip(requests, full, partial):
            pages = r.own_pages[:n]
            self.allocator.share(pages)
            forks.append(Request(list(r.prefix_pages), r.prefix_len, pages + ([next(copies)] if cut else []), r.length))
        return forks

    def truncate(self, request: Request, length: int) -> None:
        """Cut the request back to its first ``length`` tokens: the pages behind
        them are freed, and a last page that is now partial and has other
        holders is replaced by a copy, since the request will write to it."""
        if not request.prefix_len <= length <= request.length:
            raise ValueError(f"length {length} is outside [{request.prefix_len}, {request.length}], the request's "
                             "own tokens")
        keep = -(-(length - request.prefix_len) // self.page_size)
        last = request.own_pages[keep - 1] if keep and length % self.page_size else None
        pages = request.own_pages[:keep]
        if last is not None and self.allocator.holders(last) > 1:
            copy = self.allocator.allocate(1)
            try:
                self.copy_pages([last], copy)
            except Exception:
                self.allocator.free(copy)
                raise
            self.allocator.free([last])
            pages[-1:] = copy
        self.allocator.free(request.own_pages[keep:])
        request.own_pages = pages
        request.length = length

    def compact(self, requests: Sequence[Request]) -> dict[int, int]:
        """Move the requests' pages to the lowest free ids; returns the moves (old id -> new id).

        ``requests`` names every request that lists a page of theirs, as its own
        or as a prefix: all their lists are rewritten.  A page with a holder
        that is not among them stays.  Page tables made before hold the old ids:
        plan again, and let no step run on the old ones in between."""
        requests = list({id(r): r for r in requests}.values())
        held: dict[int, int] = {}
        for r in requests:
            for p in r.own_pages:
                held[p] = held.get(p, 0) + 1
        pages = sorted((p for p, n in held.items() if n == self.allocator.holders(p)), reverse=True)
        moved = {p: f for p, f in zip(pages, sorted(self.allocator._free)) if f < p}
        if moved:
            self.copy_pages(list(moved), list(moved.values()))
            self.allocator.move(moved)
            for r in requests:
                r.own_pages = [moved.get(p, p) for p in r.own_pages]
                r.prefix_pages = [moved.get(p, p) for p in r.prefix_pages]
        return moved

    def tables(self, requests) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """int32 (indptr, indices, last_page_len) for the batch."""
        return pack_rows([r.spans(self.page_size) for r in requests], self.page_size)
