"""Who holds which page of the key/value pool: the host's side of the paged cache.

The reference gives each request of a step its own run of pages (kv_cache.py:1-40, a page list and a
ring position per request). :class:`PagePool` keeps the same pool -- ``[pages + 1, 2, layers, 128, heads,
128]``, the last page the null page that unused table entries name -- for requests that come, grow,
fork, shrink and go: pages are counted by holder, a fork shares them and copies only what both sides
would write, and the rows that a request gives up are compacted away. The page contents move on the
GPU (``ops.copy_pages``, ``ops.compact_rows``); the tables are plain host lists, and :meth:`PagePool.lut`
makes the device table that ``ops.paged_chunk_attention`` and ``ops.paged_decode_attention`` read.
Everything is enqueued on the current stream, in order with the attention calls on it; a pool used on
several streams needs the caller's own ordering between them.
"""

from __future__ import annotations

from collections.abc import Hashable, Sequence

import torch

from . import ops

PAGE_ROWS = 128  # kv_cache.py: rows of a page
HEAD_DIM = 128


class PoolFullError(RuntimeError):
    """No page is free. Nothing was changed by the call that raised it."""


class PagePool:
    """``pages`` pages for ``layers`` layers of ``heads`` KV heads, fp32 or bf16. ``pool`` is the tensor."""

    def __init__(self, pages: int, layers: int, heads: int, *, dtype: torch.dtype = torch.float32,
                 device: str | torch.device = "cuda", pool: torch.Tensor | None = None):
        if pages < 1 or layers < 1 or heads < 1:
            raise ValueError(f"PagePool: pages, layers and heads must be >= 1, got {pages}, {layers}, {heads}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"PagePool: the pool is fp32 or bf16, got {dtype}")
        shape = (pages + 1, 2, layers, PAGE_ROWS, heads, HEAD_DIM)
        if pool is None:
            pool = torch.zeros(shape, dtype=dtype, device=device)
        if tuple(pool.shape) != shape or pool.dtype != dtype or not pool.is_contiguous():
            raise ValueError(f"PagePool: pool must be a contiguous {dtype} tensor of shape {shape}")
        self.pool, self.pages, self.null_page = pool, int(pages), int(pages)
        self._free = list(range(pages - 1, -1, -1))  # taken from the end: the lowest page first
        self._holders = [0] * pages
        self._tables: dict[Hashable, list[int]] = {}
        self._rows: dict[Hashable, int] = {}

    # ---- what is held ------------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def rows(self, request: Hashable) -> int:
        return self._rows[self._known(request)]

    def table(self, request: Hashable) -> list[int]:
        return list(self._tables[self._known(request)])

    def lut(self, requests: Sequence[Hashable], cols: int | None = None) -> torch.Tensor:
        """The requests' page ids, int32 ``[B, cols]`` on the device (unused entries: the null page)."""
        tables = [self._tables[self._known(r)] for r in requests]
        most = max((len(t) for t in tables), default=0)
        cols = max(1, most) if cols is None else cols
        if cols < most:
            raise ValueError(f"PagePool: a request holds {most} pages, the table has {cols} columns")
        return self._device([t + [self.null_page] * (cols - len(t)) for t in tables]).reshape(len(tables), cols)

    # ---- requests ----------------------------------------------------------------------------
    def add(self, request: Hashable, rows: int = 0) -> None:
        """A new request with room for ``rows`` rows (counted as held: the caller stores them)."""
        if request in self._tables:
            raise ValueError(f"PagePool: request {request!r} is already there")
        if rows < 0:
            raise ValueError(f"PagePool: rows must be >= 0, got {rows}")
        self._tables[request] = self._take(-(-rows // PAGE_ROWS))
        self._rows[request] = rows

    def extend(self, request: Hashable, rows: int) -> int:
        """Room for ``rows`` more rows; returns the first of them (``start`` of the chunk that stores them)."""
        start = self._rows[self._known(request)]
        if rows < 0:
            raise ValueError(f"PagePool: rows must be >= 0, got {rows}")
        table = self._tables[request]
        more = -(-(start + rows) // PAGE_ROWS) - len(table)
        shared = self._shared(request, start) if rows else []
        if more + len(shared) > len(self._free):
            raise PoolFullError(f"PagePool: {more + len(shared)} pages needed, {len(self._free)} free")
        self._own(request, shared)
        table += self._take(more)
        self._rows[request] = start + rows
        return start

    def fork(self, request: Hashable, child: Hashable) -> None:
        """``child`` holds the same rows as ``request``: full pages are shared, a partly filled last page
        is copied, so that both may append."""
        table, rows = self._tables[self._known(request)], self._rows[request]
        if child in self._tables:
            raise ValueError(f"PagePool: request {child!r} is already there")
        full = rows // PAGE_ROWS
        tail = table[full: -(-rows // PAGE_ROWS)]
        fresh = self._take(len(tail))
        for page in table[:full]:
            self._holders[page] += 1
        self._tables[child] = table[:full] + fresh
        self._rows[child] = rows
        self._copy(tail, fresh, [rows % PAGE_ROWS] * len(tail))

    def make_writable(self, request: Hashable, first_row: int) -> None:
        """Own copies of the shared pages that hold rows from ``first_row`` on (rows about to be
        overwritten in place, as the ring of the sliding window is)."""
        shared = self._shared(request, first_row)
        if len(shared) > len(self._free):
            raise PoolFullError(f"PagePool: {len(shared)} pages needed, {len(self._free)} free")
        self._own(request, shared)

    def keep(self, request: Hashable, rows: Sequence[int]) -> None:
        """Only the given rows (strictly ascending) stay, as rows 0, 1, ...; the pages that this frees are
        given back. In place where the request holds its pages alone; shared pages that would change
        are replaced by fresh ones."""
        table, have = self._tables[self._known(request)], self._rows[request]
        rows = [int(r) for r in rows]
        if any(b <= a for a, b in zip(rows, rows[1:])) or (rows and not 0 <= rows[0] <= rows[-1] < have):
            raise ValueError(f"PagePool: rows to keep must ascend strictly within 0..{have - 1}")
        cols = -(-len(rows) // PAGE_ROWS)
        same = next((i for i, r in enumerate(rows) if r != i), len(rows))  # rows that stay where they are
        first = same // PAGE_ROWS
        # With one changing page in other hands all changing pages move to fresh ones: a page that
        # is written in place must not be read later by way of another column's fresh copy.
        moved = list(range(first, cols)) if any(self._holders[p] > 1 for p in table[first:cols]) and same < len(rows) else []
        fresh = self._take(len(moved))
        to = table[:cols]
        for c, page in zip(moved, fresh):
            to[c] = page
        if same < len(rows):
            # rows below the first changing page are not listed: a fresh table column starts at `first`
            begin = first * PAGE_ROWS
            ops.compact_rows(self.pool, self._device([[*table[first:]]]),
                             self._device([to[first:]]), self._device([[r - begin for r in rows[begin:]]]),
                             self._device([len(rows) - begin]))
        self._tables[request], self._rows[request] = to, len(rows)
        self._give([p for c, p in enumerate(table) if c >= cols or to[c] != p])

    def free(self, request: Hashable) -> None:
        """The request goes; pages that no other request holds are free again."""
        self._give(self._tables.pop(self._known(request)))
        del self._rows[request]

    def defragment(self) -> int:
        """The held pages moved to the front of the pool (contents and tables); returns how many there
        are, so that pages from there on are free."""
        held = [p for p in range(self.pages) if self._holders[p]]
        n = len(held)
        src = [p for p in held if p >= n]
        dst = [p for p in range(n) if not self._holders[p]]
        self._copy(src, dst, None)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        for table in self._tables.values():
            table[:] = [to.get(p, p) for p in table]
        self._free = list(range(self.pages - 1, n - 1, -1))
        return n

    # ---- inner ---------------------------------------------------------------------------------
    def _known(self, request: Hashable) -> Hashable:
        if request not in self._tables:
            raise KeyError(f"PagePool: no request {request!r}")
        return request

    def _device(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.pool.device)

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise PoolFullError(f"PagePool: {n} pages needed, {len(self._free)} free")
        pages = [self._free.pop() for _ in range(max(0, n))]
        for p in pages:
            self._holders[p] = 1
        return pages

    def _give(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._holders[p] -= 1
            if not self._holders[p]:
                self._free.append(p)
        self._free.sort(reverse=True)

    def _shared(self, request: Hashable, first_row: int) -> list[int]:
        table = self._tables[self._known(request)]
        return [c for c in range(max(0, first_row) // PAGE_ROWS, len(table)) if self._holders[table[c]] > 1]

    def _own(self, request: Hashable, cols: Sequence[int]) -> None:
        table = self._tables[request]
        fresh = self._take(len(cols))
        old = [table[c] for c in cols]
        for c, p in zip(cols, fresh):
            table[c] = p
        self._copy(old, fresh, None)
        self._give(old)

    def _copy(self, src: Sequence[int], dst: Sequence[int], rows: Sequence[int] | None) -> None:
        if src:
            ops.copy_pages(self.pool, self._device(list(src)), self._device(list(dst)),
                           rows=None if rows is None else self._device(list(rows)))
