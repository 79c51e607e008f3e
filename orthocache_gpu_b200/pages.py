"""Pages of a cache: forking, reserving, freeing, compacting and copying, on the device.

State is three int32 tensors: ``block_tables`` (num_seqs, max_blocks), page
ids in order and -1 where a row holds none; ``seq_lens`` (num_seqs,); and
``refcounts`` (num_pages,), how many table entries name each page (0: free).
Sequences that share a history share its pages; a page is copied only when
one of its holders is about to write to it.  Nothing synchronises with the
host, and which page is handed out never depends on timing.
:class:`PagedKVCache` keeps the state of a model together.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page src[i] to dst[i] in every cache (num_pages, ...), in one launch per 128 caches.

    A negative id skips the pair; no dst may be the src or dst of another pair.
    """
    _lib.require_binding().copy_pages(caches, src, dst)


def fork_sequences(block_tables: torch.Tensor, seq_lens: torch.Tensor, refcounts: torch.Tensor, source: torch.Tensor,
                   block_size: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """New (block_tables, seq_lens, refcounts) in which row i is sequence source[i], all rows at once.

    source[i] == i keeps a row with all that it holds; another row's tokens are shared, page by page
    (the unfilled last one too: :func:`reserve_pages` copies it before a write); a negative source frees
    the row.  Reordering of beams, forks for sampling, and the end of a sequence are all this call.
    """
    return _lib.require_binding().fork_sequences(block_tables, seq_lens, refcounts, source, block_size)


def reserve_pages(caches: Sequence[torch.Tensor], block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  refcounts: torch.Tensor, wanted: torch.Tensor, block_size: int, *,
                  return_done: bool = False) -> Optional[torch.Tensor]:
    """Make room, in place, for sequence i to grow to wanted[i] tokens.

    Where a row grows and its unfilled last page has other holders, the page is copied in every cache;
    if all its holders grow, the last of them keeps it.  A row may have been shortened since the last call:
    the pages that it still holds behind its tokens are used again, and those of them that others hold are
    replaced, without a copy.  The k-th page needed (by row, then column) is the k-th lowest free one.  All
    or nothing: if free pages or table columns do not suffice, nothing changes and the device's status word is
    set.  Rows must not be written to then, as their pages may still be shared: check the word
    (:func:`check_status`) first, or, where the host must not wait, take what ``return_done`` returns, a tensor
    of one int32 on the device (1: reserved, 0: not), and let nothing grow where it is 0.
    ``seq_lens`` does not change.
    """
    return _lib.require_binding().reserve_pages(caches, block_tables, seq_lens, refcounts, wanted, block_size,
                                                return_done)


def compact_pages(caches: Sequence[torch.Tensor], block_tables: torch.Tensor,
                  refcounts: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Move the n pages in use to ids [0, n); returns the new (block_tables, refcounts).

    Cache contents move in place: the k-th used page at or above n goes to the k-th free one below it, so
    pages already below n stay.
    """
    return _lib.require_binding().compact_pages(caches, block_tables, refcounts)


class PagedKVCache:
    """The paged key and value caches of every layer, with their tables.

    ``k[layer]`` / ``v[layer]`` are (num_pages, kv_heads, block_size, head_dim).  Rows of the tables are
    the sequences of a batch; a row with length 0 and no pages is idle.  :meth:`fork`, :meth:`free` and
    :meth:`compact` put new tensors in the place of the tables, so a captured graph that read the old ones has
    to be captured again; :meth:`reserve` and the appends work in place.
    """

    def __init__(self, layers: int, num_pages: int, kv_heads: int, head_dim: int, *, max_seqs: int, max_tokens: int,
                 block_size: int = 16, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if block_size < 1 or block_size & (block_size - 1):
            raise ValueError(f"block_size ({block_size}) must be a power of 2")
        self.block_size = block_size
        shape = (num_pages, kv_heads, block_size, head_dim)
        self.k: List[torch.Tensor] = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v: List[torch.Tensor] = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.block_tables = torch.full((max_seqs, -(-max_tokens // block_size)), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.refcounts = torch.zeros(num_pages, dtype=torch.int32, device=device)

    @property
    def caches(self) -> List[torch.Tensor]:
        return self.k + self.v

    def fork(self, source: torch.Tensor) -> None:
        """Row i becomes a copy of row source[i] (shared pages); a negative source frees it."""
        self.block_tables, self.seq_lens, self.refcounts = fork_sequences(
            self.block_tables, self.seq_lens, self.refcounts, source, self.block_size)

    def free(self, rows: Sequence[int]) -> None:
        """End the sequences in ``rows``."""
        source = torch.arange(self.seq_lens.numel(), dtype=torch.int32)
        source[list(rows)] = -1
        self.fork(source.to(self.seq_lens.device))

    def reserve(self, tokens: torch.Tensor, check: bool = True) -> Optional[torch.Tensor]:
        """Make room for tokens[i] more tokens in row i; with ``check``, raise if there are too few pages.

        Without ``check`` the host does not wait, and a tensor of one int32 comes back: 1, or 0 if there are too
        few pages, in which case no row may be written to.
        """
        done = reserve_pages(self.caches, self.block_tables, self.seq_lens, self.refcounts, self.seq_lens + tokens,
                             self.block_size, return_done=not check)
        if check:
            _lib.check_status(self.seq_lens.device)
        return done

    def compact(self) -> None:
        """Move the pages in use to the lowest ids."""
        self.block_tables, self.refcounts = compact_pages(self.caches, self.block_tables, self.refcounts)

    def free_pages(self) -> int:
        """Number of free pages (synchronises)."""
        return int((self.refcounts == 0).sum())
