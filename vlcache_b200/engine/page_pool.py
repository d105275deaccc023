"""Which pages of a paged KV cache are in use, by how many requests: allocate, fork, free, compact.

Host bookkeeping over page numbers; the copies it asks for run in one launch per call for all
layers (``engine.kv_cache.copy_pages``, vlc_copy_pages), over either cache format.  Block
tables are the lists of page numbers that the metadata builders take.  A forked request
(several answers to one prompt, a search's branches) shares its full pages; the last page,
which both sides will write, is copied.  Compaction moves the used pages to the front of the
pool, so that its tail can be given back or handed to another cache.
"""
from __future__ import annotations

from collections import deque

import numpy as np

from .kv_cache import BLOCK_SIZE


class PagePool:
    """Pages ``0 .. num_pages - 1`` with the number of block tables that hold each."""

    def __init__(self, num_pages: int, block_size: int = BLOCK_SIZE):
        if num_pages <= 0 or block_size <= 0:
            raise ValueError("num_pages and block_size must be positive")
        self.num_pages = num_pages
        self.block_size = block_size
        self.refs = [0] * num_pages
        self.free_pages = deque(range(num_pages))

    @property
    def num_free(self) -> int:
        return len(self.free_pages)

    def pages_for(self, num_tokens: int) -> int:
        return (num_tokens + self.block_size - 1) // self.block_size

    def allocate(self, num_pages: int) -> list[int] | None:
        """``num_pages`` fresh pages, or None (and no change) when fewer are free."""
        if num_pages < 0:
            raise ValueError("num_pages must not be negative")
        if num_pages > len(self.free_pages):
            return None
        pages = [self.free_pages.popleft() for _ in range(num_pages)]
        for p in pages:
            self.refs[p] = 1
        return pages

    def _check_live(self, pages) -> None:
        for p in pages:
            if not 0 <= p < self.num_pages or self.refs[p] <= 0:
                raise ValueError(f"page {p} is not in use")

    def fork(self, block_table: list[int], num_tokens: int) -> tuple[list[int], list[tuple[int, int]]] | None:
        """A second block table for the same ``num_tokens`` tokens: full pages shared, a part-filled
        last page copied.  Returns (table, [(source, destination)] to copy before either side
        writes), or None (and no change) when no page is free for the copy."""
        used = self.pages_for(num_tokens)
        if num_tokens < 0 or used > len(block_table):
            raise ValueError("the block table does not hold that many tokens")
        self._check_live(block_table[:used])
        full = num_tokens // self.block_size
        table, copies = list(block_table[:full]), []
        if used > full:
            fresh = self.allocate(1)
            if fresh is None:
                return None
            copies.append((block_table[full], fresh[0]))
            table += fresh
        for p in block_table[:full]:
            self.refs[p] += 1
        return table, copies

    def free(self, block_table: list[int]) -> None:
        """Give a block table's pages back; a page is free once no table holds it."""
        count: dict[int, int] = {}
        for p in block_table:
            count[p] = count.get(p, 0) + 1
        for p, n in count.items():
            if not 0 <= p < self.num_pages or self.refs[p] < n:
                raise ValueError(f"page {p} is freed more often than it is held")
        for p, n in count.items():
            self.refs[p] -= n
            if self.refs[p] == 0:
                self.free_pages.append(p)

    def compact(self) -> tuple[list[int], list[int], np.ndarray]:
        """Move the used pages to ``0 .. used - 1``.  Returns (sources, destinations, page map):
        the copies to make (``copy_pages``), and the int32 map that every block table has to
        go through (``remap``, or ``ops.remap_block_tables`` for one on the device)."""
        used = self.num_pages - len(self.free_pages)
        holes = [p for p in range(used) if self.refs[p] == 0]
        src = [p for p in range(used, self.num_pages) if self.refs[p] > 0]
        dst = holes[:len(src)]
        page_map = np.arange(self.num_pages, dtype=np.int32)
        for s, d in zip(src, dst):
            page_map[s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.free_pages = deque(range(used, self.num_pages))
        return src, dst, page_map


def remap(block_table: list[int], page_map: np.ndarray) -> list[int]:
    """A host block table after ``PagePool.compact``; entries of -1 (padding) stay, as on the device."""
    for p in block_table:
        if not -1 <= p < len(page_map):
            raise ValueError(f"page {p} is outside the pool's {len(page_map)}")
    return [int(page_map[p]) if p >= 0 else -1 for p in block_table]
