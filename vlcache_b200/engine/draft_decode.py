"""Decode steps of several tokens a sequence (drafted tokens to verify), kept on the device.

A step of every running sequence takes its last sampled token and K drafted ones: ``begin`` takes
pages and makes positions and slots (vlc_step_metadata), the model runs its layers over the
[places * (K + 1)] rows (``Attention.forward`` scatters and attends, with the layer's sliding
window), and ``finish`` verifies the drafts and moves the lengths on (vlc_verify_drafts).  Nothing is
read back in between, so a step can be captured into a graph and replayed; the host looks at the
emitted tokens whenever it wants to.

Pages come from a ``PagePool``: ``lend`` moves some to the device's free list, which the steps take
pages from and give those behind the window back to; ``settle`` returns them.  A sequence enters with
the block table that its prompt was stored through (``admit``) and leaves with ``retire``.  The
tables own their pages: a forked table, which shares some, cannot enter.  After ``PagePool.compact``
``block_tables`` and ``free_pages.view(1, -1)`` go through ``ops.remap_block_tables`` as every device table does.
"""
from __future__ import annotations

import torch

from .. import ops
from ..utils.context import set_context
from .page_pool import PagePool


class DraftDecode:
    """``places`` sequences of up to ``max_pages`` pages each, ``num_drafts`` drafted tokens a step.
    ``window`` / ``sinks``: the model's sliding window and first visible tokens where every layer has
    it (pages behind it are given back); 0 where some layer sees all keys."""

    def __init__(self, pool: PagePool, places: int, max_pages: int, num_drafts: int, window: int = 0, sinks: int = 0,
                 device: torch.device | str = "cuda"):
        if not 0 < places <= 65535 or max_pages <= 0 or not 0 <= num_drafts <= 31:
            raise ValueError("places: 1 .. 65535, max_pages: positive, num_drafts: 0 .. 31")
        if pool.block_size % 32:
            raise ValueError("block_size must be a multiple of 32")
        self.pool, self.places, self.max_pages = pool, places, max_pages
        self.num_tokens = num_drafts + 1
        self.window, self.sinks = int(window), int(sinks)
        i32 = dict(dtype=torch.int32, device=device)
        self.context_lens = torch.full((places,), -1, **i32)   # tokens in the cache; below 0: an idle place
        self.block_tables = torch.full((places, max_pages), -1, **i32)
        self.free_pages = torch.full((pool.num_pages,), -1, **i32)
        self.num_free = torch.zeros(1, **i32)
        self.new_lens = torch.full((places,), self.num_tokens, **i32)

    # ---- the host's side: pages and sequences come and go (device reads and writes: not for graph capture)
    def lend(self, num_pages: int) -> bool:
        """Move ``num_pages`` pages of the pool to the device's free list; False (and no change) when fewer are free."""
        pages = self.pool.allocate(num_pages)
        if pages is None:
            return False
        self._put(pages)
        return True

    def _put(self, pages: list[int]) -> None:
        count = int(self.num_free)
        if pages:
            self.free_pages[count:count + len(pages)] = torch.tensor(pages, dtype=torch.int32).to(self.free_pages.device)
        self.num_free.fill_(count + len(pages))

    def settle(self) -> None:
        """Give the free list's pages back to the pool."""
        count = int(self.num_free)
        self.pool.free(self.free_pages[:count].tolist())
        self.num_free.zero_()

    def admit(self, place: int, block_table: list[int], num_tokens: int) -> None:
        """A sequence of ``num_tokens`` tokens in the cache, stored through ``block_table`` (its pages are the
        decoder's from here on), takes an idle place.  Its next token, not in the cache yet, is the
        first of its rows in the next step.  Entries of pages that it no longer sees, behind the window and the sinks,
        may be -1."""
        if not 0 <= place < self.places:
            raise ValueError(f"place {place} is outside the {self.places}")
        if int(self.context_lens[place]) >= 0:
            raise ValueError(f"place {place} is taken")
        if num_tokens < 0 or self.pool.pages_for(num_tokens) > len(block_table):
            raise ValueError("the block table does not hold that many tokens")
        if len(block_table) > self.max_pages:
            raise ValueError(f"a block table of {len(block_table)} pages, {self.max_pages} at most")
        gone = [p == -1 and self._behind(i, num_tokens) for i, p in enumerate(block_table)]
        pages = [p for p, g in zip(block_table, gone) if not g]
        shared = [p for p in pages if not 0 <= p < self.pool.num_pages or self.pool.refs[p] != 1]
        if shared:
            raise ValueError(f"page {shared[0]} is not this table's alone")
        if len(set(pages)) != len(pages):
            raise ValueError("a page is in the block table twice")
        mine = torch.cat((self.block_tables.flatten(), self.free_pages[:int(self.num_free)]))
        if pages and bool(torch.isin(torch.tensor(pages, dtype=torch.int32).to(mine.device), mine).any()):
            raise ValueError("a page is in another place's table or was lent")
        row = torch.full((self.max_pages,), -1, dtype=torch.int32)
        row[:len(block_table)] = torch.tensor(block_table, dtype=torch.int32)
        self.block_tables[place] = row.to(self.block_tables.device)
        self.context_lens[place] = num_tokens

    def _behind(self, page: int, num_tokens: int) -> bool:
        """Whether entry ``page`` of a table is one that no row at position ``num_tokens`` or later sees."""
        block = self.pool.block_size
        return self.window > 0 and page * block >= self.sinks and (page + 1) * block <= num_tokens - self.window + 1

    def retire(self, place: int) -> int:
        """A sequence leaves: its pages go back to the pool, its place is idle.  Returns its tokens in the cache."""
        if not 0 <= place < self.places:
            raise ValueError(f"place {place} is outside the {self.places}")
        tokens = int(self.context_lens[place])
        if tokens < 0:
            raise ValueError(f"place {place} is idle")
        self.pool.free([p for p in self.block_tables[place].tolist() if p >= 0])
        self.block_tables[place] = -1
        self.context_lens[place] = -1
        return tokens

    # ---- a step, on the device
    def begin(self) -> torch.Tensor:
        """Take the step's pages, make its metadata and install it (``set_context``); returns the rows'
        positions int64 [places * (num_drafts + 1)].  The rows are the places' tokens, one place behind
        another: its last token, then its drafts; idle places have rows too, which nothing is stored for.
        A rotary with several axes, whose positions behind an image differ from the tokens' numbers by an offset of
        each sequence, takes ``(positions.view(places, -1) + offsets.view(-1, 1)).view(1, -1).expand(axes, -1)``,
        ``offsets`` int64 [places] on the device (0 in idle places)."""
        rows = self.places * self.num_tokens
        positions, slots, _, _, lens = ops.step_metadata(self.context_lens, self.new_lens, self.block_tables,
                                                         self.free_pages, self.num_free, self.pool.block_size, rows,
                                                         self.window, self.sinks)
        # The bound takes in a step that reaches past a table's end (cut lengths would move the rows before the end), but
        # no more: a step that begins there is cut, none of whose rows count, so that a sequence's single token stays in
        # its table (vlc_decode_attn has no width to look at).
        set_context(False, slot_mapping=slots, context_lens=lens, block_tables=self.block_tables,
                    max_context_len=self.max_pages * self.pool.block_size + self.num_tokens - 1, num_tokens=self.num_tokens)
        return positions

    def finish(self, drafts: torch.Tensor, target_probs: torch.Tensor, draft_probs: torch.Tensor | None,
               u: torch.Tensor, u_last: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Verify the step's drafts (``ops.verify_drafts``; int64 [places, num_drafts], -1 where a place
        has fewer) and keep what was accepted: the lengths move on by emitted.  Returns (tokens, emitted);
        of a place's tokens the last is its next step's first row.  A place that found no page for some of its rows
        (the free list ran out, or its table ended: ``ops.device_error``) has no drafts from there on; one that found
        none for its first row emits nothing (emitted 0, tokens -1) and begins its next step with the same
        token, when pages were lent."""
        if drafts.shape != (self.places, self.num_tokens - 1):
            raise ValueError(f"drafts: [{self.places}, {self.num_tokens - 1}]")
        return ops.verify_drafts(drafts, target_probs, draft_probs, u, u_last, self.context_lens, self.block_tables,
                                 self.pool.block_size)
