"""A key-value cache in pages for serving many sequences at once (no counterpart in the
reference, whose cache holds one batch of equal lengths: nn/transformer.py:49-66).

:class:`PagedKVCache` owns one pool of key pages and one of value pages for all layers and
keeps the books on the host: which pages a sequence's positions lie on, how many sequences
share a page, which pages are free. Forking a sequence shares its pages; a shared page is
copied when one of its owners is about to write to it. Compaction moves the pages in use to
the front of the pools, so that :meth:`PagedKVCache.resize` can give the rest back.

    cache = model.make_paged_cache(num_pages=512)
    a = cache.add()
    model(prompt[None], cache=cache.batch([a]))       # prefill: any number of tokens
    b = cache.fork(a)                                 # shares the prompt's pages
    logits = model(next_ids[:, None], cache=cache.batch([a, b]))
"""

from __future__ import annotations

import heapq
from collections.abc import Sequence
from dataclasses import dataclass, field
from typing import Any

import numpy as np

from tensorgrad_b200 import device
from tensorgrad_b200.device import DeviceArray
from tensorgrad_b200.ops.paged import copy_pages
from tensorgrad_b200.ops.shape import strided_copy
from tensorgrad_b200.tensor import Tensor, get_default_dtype

__all__ = ["PagedBatch", "PagedKVCache"]


@dataclass
class _Held:
    """One sequence: its pages in order and the positions it holds on them."""

    pages: list[int] = field(default_factory=list)
    length: int = 0


class PagedKVCache:
    """Pools ``(layers, num_pages, kv_heads, page_size, head_dim)`` of keys and values, and
    the sequences on them (see the module's docstring). Sequences are named by the integers
    that :meth:`add` and :meth:`fork` return."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int = 16, dtype: Any = None) -> None:
        for name, n in (("layers", layers), ("kv_heads", kv_heads), ("head_dim", head_dim),
                        ("num_pages", num_pages), ("page_size", page_size)):
            if n <= 0:
                raise ValueError(f"{name} must be positive, got {n}")
        self.page_size, self.num_pages = page_size, num_pages
        self._dtype = np.dtype(get_default_dtype() if dtype is None else dtype)
        self._shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self._pools: tuple[Tensor, Tensor] | None = None
        self._refs = np.zeros(num_pages, dtype=np.int64)
        self._free = list(range(num_pages))  # a heap: the lowest page first
        self._held: dict[int, _Held] = {}
        self._next = 0

    # ------------------------------------------------------------------ storage
    @property
    def keys(self) -> Tensor:
        return self._storage()[0]

    @property
    def values(self) -> Tensor:
        return self._storage()[1]

    def _storage(self) -> tuple[Tensor, Tensor]:
        if self._pools is None:
            self._pools = self._allocate(self._shape)
        return self._pools

    def _allocate(self, shape: tuple[int, ...]) -> tuple[Tensor, Tensor]:
        return (Tensor._wrap(device.empty(shape, self._dtype)),
                Tensor._wrap(device.empty(shape, self._dtype)))

    def layer(self, index: int) -> tuple[DeviceArray, DeviceArray]:
        """One layer's pools ``(num_pages, kv_heads, page_size, head_dim)``, as views."""
        one = self._shape[1:]
        n = int(np.prod(one))
        return (self.keys.data.flat_view(index * n, n, one),
                self.values.data.flat_view(index * n, n, one))

    @property
    def pages_in_use(self) -> int:
        return self.num_pages - len(self._free)

    # ------------------------------------------------------------------ sequences
    def _get(self, seq: int) -> _Held:
        try:
            return self._held[seq]
        except KeyError:
            raise KeyError(f"no sequence {seq} in the cache") from None

    def length(self, seq: int) -> int:
        """Positions the sequence holds."""
        return self._get(seq).length

    def pages(self, seq: int) -> tuple[int, ...]:
        """The sequence's pages in order."""
        return tuple(self._get(seq).pages)

    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._held[seq] = _Held()
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence that continues from ``seq``'s positions, sharing its pages."""
        old = self._get(seq)
        used = old.pages[:-(-old.length // self.page_size)]
        new = self.add()
        self._held[new] = _Held(list(used), old.length)
        for p in used:
            self._refs[p] += 1
        return new

    def free(self, seq: int) -> None:
        """Drop a sequence; pages that no other sequence shares become free."""
        for p in self._get(seq).pages:
            self._release(p)
        del self._held[seq]

    def _release(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def reserve(self, seqs: Sequence[int], tokens: int) -> None:
        """Make room for ``tokens`` more positions of every sequence: pages are added, and a
        page about to be written that other sequences share is copied. ``MemoryError`` (and
        nothing changed) where the pool has too few free pages."""
        held = [self._get(s) for s in seqs]
        if len(set(seqs)) != len(held):
            raise ValueError(f"a sequence is named twice in {list(seqs)}")
        if tokens < 0:
            raise ValueError(f"cannot reserve {tokens} positions")
        if tokens == 0:
            return
        size = self.page_size
        # The pages that will be written: from the one the next position lies on.
        refs = self._refs.copy()
        shared: list[tuple[_Held, int]] = []
        grow = 0
        for h in held:
            for i in range(h.length // size, len(h.pages)):
                if refs[h.pages[i]] > 1:  # the last owner left to write keeps the page
                    refs[h.pages[i]] -= 1
                    shared.append((h, i))
            grow += max(0, -(-(h.length + tokens) // size) - len(h.pages))
        if len(shared) + grow > len(self._free):
            raise MemoryError(f"paged cache: {len(shared) + grow} more pages needed, "
                              f"{len(self._free)} of {self.num_pages} free")
        src, dst = [], []
        for h, i in shared:
            new = self._take()
            if i * size < h.length:
                src.append(h.pages[i])
                dst.append(new)
            self._release(h.pages[i])
            h.pages[i] = new
        for h in held:
            while len(h.pages) * size < h.length + tokens:
                h.pages.append(self._take())
        if src:
            copy_pages(self.keys, self.values, src, dst)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    # ------------------------------------------------------------------ memory
    def compact(self) -> int:
        """Move the pages in use to the front of the pools; returns how many there are (the
        smallest ``num_pages`` that :meth:`resize` takes). Spare pages that were reserved but
        hold no positions are given up first."""
        for h in self._held.values():
            keep = -(-h.length // self.page_size)
            for p in h.pages[keep:]:
                self._release(p)
            del h.pages[keep:]
        used = self.pages_in_use
        live = np.flatnonzero(self._refs)
        src = live[live >= used]
        dst = np.flatnonzero(self._refs[:used] == 0)
        if src.size:
            copy_pages(self.keys, self.values, src, dst)
            to = np.arange(self.num_pages)
            to[src] = dst
            for h in self._held.values():
                h.pages = to[h.pages].tolist()
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
        self._free = list(range(used, self.num_pages))
        return used

    def resize(self, num_pages: int) -> None:
        """Pools of ``num_pages`` pages: grown, or (compacted first) shrunk."""
        if num_pages <= 0:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        if num_pages < self.num_pages:
            used = self.compact()
            if used > num_pages:
                raise ValueError(f"{used} pages are in use, more than {num_pages}")
        kept = min(num_pages, self.num_pages)
        shape = (self._shape[0], num_pages, *self._shape[2:])
        if self._pools is not None:
            pools = self._allocate(shape)
            for old, new in zip(self._pools, pools, strict=True):
                self._carry(old, new, kept)
            self._pools = pools
        self._shape, self.num_pages = shape, num_pages
        refs = np.zeros(num_pages, dtype=np.int64)
        refs[:kept] = self._refs[:kept]
        self._refs = refs
        self._free = np.flatnonzero(refs == 0).tolist()

    def _carry(self, old: Tensor, new: Tensor, pages: int) -> None:
        """The first ``pages`` pages of every layer from one pool to another."""
        n = int(np.prod(self._shape[2:]))
        strided_copy(old.data.ptr, [old.shape[1] * n, 1], new.data.ptr, [new.shape[1] * n, 1],
                     (self._shape[0], pages * n), self._dtype.itemsize)

    def batch(self, seqs: Sequence[int]) -> PagedBatch:
        """The sequences of one model call, in the order of its rows."""
        return PagedBatch(self, list(seqs))


class PagedBatch:
    """Rows of a model call on a :class:`PagedKVCache`: row ``i`` continues sequence
    ``seqs[i]``. Made by :meth:`PagedKVCache.batch`, consumed by ``GPT.forward``."""

    def __init__(self, cache: PagedKVCache, seqs: list[int]) -> None:
        if not seqs:
            raise ValueError("a batch names at least one sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError(f"a sequence is named twice in {seqs}")
        self.cache, self.seqs = cache, seqs
        self._starts()  # unknown sequences raise here

    def _starts(self) -> np.ndarray:
        return np.array([self.cache.length(s) for s in self.seqs], dtype=np.int64)

    @property
    def lengths(self) -> np.ndarray:
        """Positions each row's sequence holds already."""
        return self._starts()

    def check_model(self, layers: int, attn: Any, dtype: np.dtype[Any]) -> None:
        """Refuse a model whose layers, heads or type are not the cache's."""
        have = (self.cache._shape[0], self.cache._shape[2], self.cache._shape[4],
                self.cache._dtype)
        want = (layers, attn.num_heads, attn.head_dim, np.dtype(dtype)) if layers else have
        if have != want:
            raise ValueError("the paged cache holds (layers, heads, head_dim, dtype) "
                             f"{(*have[:3], str(have[3]))}, the model has "
                             f"{(*want[:3], str(want[3]))}")

    def begin(self, tokens: int) -> list[PagedLayer]:
        """Reserve ``tokens`` more positions for every row and describe the step to each
        layer. The sequences grow only with :meth:`commit`."""
        cache = self.cache
        cache.reserve(self.seqs, tokens)
        starts = self._starts()
        ends = starts + tokens
        width = max(1, -(-int(ends.max()) // cache.page_size))
        table = np.zeros((len(self.seqs), width), dtype=np.int64)
        for row, seq in enumerate(self.seqs):
            ids = cache.pages(seq)[:width]
            table[row, :len(ids)] = ids
        # One upload for the table and both length vectors.
        both = device.from_numpy(np.concatenate([table.reshape(-1), starts, ends]))
        n = table.size
        on_device = (both.flat_view(0, n, table.shape), both.flat_view(n, len(starts)),
                     both.flat_view(n + len(starts), len(ends)))
        return [PagedLayer(*cache.layer(i), *on_device, starts, tokens)
                for i in range(cache._shape[0])]

    def commit(self, tokens: int) -> None:
        """The step's positions have been written: the sequences grow by ``tokens``."""
        for s in self.seqs:
            self.cache._get(s).length += tokens


@dataclass
class PagedLayer:
    """One layer's pools and one step's page table, with the sequences' lengths before the
    step (``starts``, also on the host) and after it (``ends``)."""

    keys: DeviceArray
    values: DeviceArray
    table: DeviceArray
    starts: DeviceArray
    ends: DeviceArray
    host_starts: np.ndarray
    tokens: int
