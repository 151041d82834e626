"""Host side of a paged KV cache: which pages of a pool each sequence holds.

The pages themselves are device memory of the engine (KVCache::reservePaged) or
of dli_sm100.paged_kv_pages; the paged operators find a sequence's rows through
its row of an int32 page table: row p lies in page table[p // page_size].
"""
from __future__ import annotations


class PagePool:
    """Hands out the pages 0 .. num_pages - 1 to sequences."""

    def __init__(self, num_pages: int, page_size: int):
        if num_pages <= 0 or page_size <= 0:
            raise ValueError("PagePool: num_pages and page_size must be positive")
        self.num_pages, self.page_size = num_pages, page_size
        self._free = list(range(num_pages - 1, -1, -1))

    @property
    def free(self) -> int:
        """Pages that no sequence holds."""
        return len(self._free)

    def pages_for(self, rows: int) -> int:
        return -(-rows // self.page_size)

    def grow(self, sequences: list[list[int]], rows: list[int]) -> None:
        """Appends pages to the lists of several sequences until they hold rows[i]
        rows each; raises MemoryError, and gives none, when the pool has too few."""
        if len(sequences) != len(rows) or any(r < 0 for r in rows):
            raise ValueError("PagePool: one non-negative row count per sequence")
        more = [max(0, self.pages_for(r) - len(p)) for p, r in zip(sequences, rows)]
        if sum(more) > self.free:
            raise MemoryError(f"page pool: {sum(more)} pages needed, {self.free} free")
        for pages, n in zip(sequences, more):
            pages.extend(self._free.pop() for _ in range(n))

    def give_back(self, pages: list[int]) -> None:
        """Returns a sequence's pages (the list is emptied)."""
        held = set(pages)
        if len(held) != len(pages) or held & set(self._free) or not held <= set(range(self.num_pages)):
            raise ValueError("PagePool: a page given back twice, or one of another pool")
        self._free.extend(reversed(pages))
        pages.clear()
