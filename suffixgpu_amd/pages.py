"""PagePool: the page tables of a paged cache, kept on the device.

After a speculative step only the device knows how long the rows are.  A pool gives
them the pages for the next step's tokens and takes back what rejected drafts and
finished requests held, without a host read.  No counterpart in the reference,
whose cache is the engine's.
"""

from __future__ import annotations

import threading

import torch

from suffixgpu_amd import _lib
from suffixgpu_amd._lib import (SuffixGPUError, check, count_arg, elsewhere,
                                lib, require_gpu, stream_of)


class PagePool:
    """``num_pages`` pages of ``page_size`` tokens (a power of two, up to 65536)
    for up to ``rows`` (4096) rows of at most ``width`` pages each.

    ``table`` [rows, width] int32 is the page table that ``KV4Cache``'s calls
    take: page ids of what a row holds, -1 behind them.  ``held`` [rows] int32 is
    how many that are, ``num_free`` [1] int32 how many no row holds.  All three
    are the pool's own, to be read; calls on one pool are ordered by their
    stream."""

    def __init__(self, num_pages: int, rows: int, width: int,
                 page_size: int = 64, device: torch.device | str = "cuda"):
        if not 1 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in 1..65536")
        if not 0 <= num_pages <= 1 << 30:
            raise ValueError("num_pages must be in 0..2^30")
        if not 1 <= rows <= _lib.PAGES_ROWS:
            raise ValueError(f"rows must be in 1..{_lib.PAGES_ROWS}")
        if not 1 <= width <= (1 << 30) // page_size:
            raise ValueError("width must be in 1..2^30 / page_size")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise SuffixGPUError("PagePool needs a ROCm GPU device; there is "
                                 "no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.num_pages = int(num_pages)
        self.rows = int(rows)
        self.width = int(width)
        self.page_size = int(page_size)
        i32 = dict(dtype=torch.int32, device=self.device)
        # page 0 on top
        self._stack = torch.arange(self.num_pages - 1, -1, -1, **i32)
        self._num_free = torch.full((1,), self.num_pages, **i32)
        self._held = torch.zeros(self.rows, **i32)
        self._table = torch.full((self.rows, self.width), -1, **i32)
        self._plan = torch.empty(3 * self.rows + 4, **i32)
        self._enqueue = threading.Lock()
        self._view = _lib.SfxPages(
            self._stack.data_ptr() or None, self._num_free.data_ptr(),
            self._held.data_ptr(), self._table.data_ptr(), self.num_pages,
            self.rows, self.width, self.page_size, self._plan.data_ptr())

    @property
    def table(self) -> torch.Tensor:
        return self._table

    @property
    def held(self) -> torch.Tensor:
        return self._held

    @property
    def num_free(self) -> torch.Tensor:
        return self._num_free

    def _lengths(self, name: str, t: torch.Tensor, n: int | None = None):
        if (t.dim() != 1 or t.device != self.device or t.shape[0] > self.rows
                or (n is not None and t.shape[0] != n)
                or t.is_floating_point() or t.dtype is torch.bool):
            require_gpu(t)
            raise ValueError(f"{name} must hold "
                             + (f"up to {self.rows}" if n is None else f"{n}")
                             + f" integers on {self.device}")
        return count_arg(t)

    def resize(self, lengths: torch.Tensor) -> torch.Tensor:
        """Rows 0 .. n - 1 hold the pages of ``lengths`` [n] tokens afterwards (at
        most ``width`` of them); a negative length leaves its row as it is, and so
        are the rows from n on.  A row that grows takes pages that were free when
        the call began, the first row first: where they run out, rows have fewer.
        A row that shrinks gives back its last pages, free from the next call on.
        Lengths put back as they were before a call put the pages back as well,
        where no row then had fewer than its length asks for.

        Returns room [n] int32: the tokens that each row's pages hold."""
        if elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.resize(lengths)
        t, is64 = self._lengths("lengths", lengths)
        n = t.shape[0]
        room = torch.empty(n, dtype=torch.int32, device=self.device)
        if n:
            # (the C call lets other threads run)
            with self._enqueue:
                rc = lib().sfx_pages_resize(self._view, t.data_ptr(), is64, n,
                                            room.data_ptr(),
                                            stream_of(self.device))
            check(rc, "PagePool.resize")
        return room

    def slots(self, start: torch.Tensor, tokens: int,
              count: torch.Tensor | None = None) -> torch.Tensor:
        """Where positions ``start[r] + i``, i < ``tokens``, of rows 0 .. n - 1
        lie: page id * page_size + position % page_size, [n, tokens] int64; -1
        where a row holds no page, for i >= ``count[r]``, and in all of a row whose
        start is negative (as one that is not in use has it).  An index into the
        tokens of a cache of such pages (``KV4Cache`` takes ``table`` itself)."""
        if elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.slots(start, tokens, count)
        s, s64 = self._lengths("start", start)
        n = s.shape[0]
        c, c64 = (None, 0) if count is None else self._lengths("count", count,
                                                               n)
        out = torch.empty(n, int(tokens), dtype=torch.int64,
                          device=self.device)
        if n and tokens:
            check(lib().sfx_pages_slots(self._view, s.data_ptr(), s64,
                                        None if c is None else c.data_ptr(),
                                        c64, n, int(tokens), out.data_ptr(),
                                        stream_of(self.device)),
                  "PagePool.slots")
        return out
