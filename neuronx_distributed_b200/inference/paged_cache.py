"""Key/value cache in pages: one pool per layer ``[pages, page_size, H_kv_local, D]``, a table of pages per batch row, and a prefix that all rows
share.  Beside ``kv_cache.py``, whose rows are contiguous and as long as the longest sequence may get, rows here hold as many pages as they need,
and what they begin alike is there once.  The pages themselves are written and read by ``ops.paged`` (``csrc/paged.cu``); this class says
whose they are.  Tables live on the device at fixed addresses (captured and recorded programs read them as they are when they run); pages are handed
out on the host, so a program takes none: its rows have to be reserved before it runs (:meth:`PagedKVCacheManager.check` says whether they were), and
the length of the shared prefix is part of it.  :class:`DevicePagedKVCacheManager` hands pages out on the device instead, so that programs take what they
need and nothing waits for positions.  Either keeps numbers of the model's type or, with ``bits=4``, codes (``ops.paged_int4``)."""
from __future__ import annotations

from contextlib import contextmanager
from typing import Iterator, List, Optional

import torch

from ..ops import page_tables, paged_int4
from ..utils.plan_registry import recording


class PagedKVCacheManager:
    def __init__(self, num_layers: int, batch_size: int, max_seq_len: int, num_kv_heads_local: int, head_dim: int, page_size: int = 32,
                 num_pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device=None, bits: Optional[int] = None):
        """``num_pages``: of the pool (default: enough for every row to be ``max_seq_len`` long).  ``bits``: 4: keys and values as codes, ``k`` and ``v``
        hold :class:`ops.paged_int4.Pages`."""
        if bits not in (None, 4):
            raise ValueError(f"keys and values are held in the model's type or in 4 bits, got {bits}")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"a page holds a multiple of 16 tokens, got {page_size}")
        self.num_layers, self.batch_size, self.max_seq_len, self.page_size = num_layers, batch_size, max_seq_len, page_size
        self.columns = (max_seq_len + page_size - 1) // page_size
        self.num_pages = batch_size * self.columns if num_pages is None else num_pages
        if self.num_pages < 1:
            raise ValueError("a pool without pages")
        shape = (self.num_pages, page_size, num_kv_heads_local, head_dim)
        self.bits = bits

        def pool():
            return torch.zeros(shape, dtype=dtype, device=device) if bits is None else paged_int4.new_pages(*shape, device=device)

        self.k: List = [pool() for _ in range(num_layers)]
        self.v: List = [pool() for _ in range(num_layers)]
        self.page_table = torch.full((batch_size, self.columns), -1, dtype=torch.int32, device=device)
        self._shared_table = torch.full((self.columns,), -1, dtype=torch.int32, device=device)
        self.shared_pages: Optional[torch.Tensor] = None      # [n] int32, the beginning of that table: what every row begins with
        self.page_table._plan_state = True                    # a launch plan keeps nothing that follows from it (inference/launch_plan.py)
        self.lost = torch.zeros(1, dtype=torch.int32, device=device)        # becomes 1 where a token had no page (ops.paged.rope_append)
        self._shared: List[int] = []
        self._rows: List[List[int]] = [[] for _ in range(batch_size)]       # pages of a row behind the shared ones
        self._free: List[int] = list(range(self.num_pages))[::-1]
        # what slots() gives ops.page_tables.assign for rows that stay as they are: no free pages, all columns to be looked at
        self._no_ring = torch.zeros(self.num_pages, dtype=torch.int32, device=device)
        self._no_span = torch.zeros(2, dtype=torch.long, device=device)
        self._ahead = False                                   # inside reserved_ahead
        self._programs: Optional[int] = None                  # shared pages that captured and recorded programs count on

    @property
    def shared_tokens(self) -> int:
        return len(self._shared) * self.page_size

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def in_program(self) -> bool:
        """A program is being captured into a CUDA graph, or recorded into a launch plan."""
        return recording() or (self.page_table.is_cuda and torch.cuda.is_current_stream_capturing())

    def note_program(self) -> None:
        """What is being captured or recorded counts on the length of the shared prefix from now on."""
        if self.in_program():
            self._programs = len(self._shared)

    def forget_programs(self) -> None:
        """The programs captured or recorded so far are not run any more."""
        self._programs = None
        self.lost.zero_()

    def check(self) -> None:
        """Raises if a captured or recorded program has run for tokens without a page since the last look: their keys are missing from what came
        after.  Waits for the device where there are such programs; sequences that end (:meth:`release`, :meth:`take_shared`) are a look, too."""
        if self._programs is not None and bool(self.lost):
            self.lost.zero_()
            raise RuntimeError("a captured or recorded program ran for tokens without a page, whose keys are lost: rows have to be reserved before it runs, "
                               f"and end at max_seq_len {self.max_seq_len}")

    def _take(self, n: int) -> List[int]:
        if n and self.in_program():
            raise RuntimeError("pages are handed out on the host: reserve them before the call is captured or recorded")
        if n > len(self._free):
            raise RuntimeError(f"the key/value pool has {len(self._free)} pages left, {n} are needed")
        return [self._free.pop() for _ in range(n)]

    def slots(self, positions: torch.Tensor, new: int, lens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Slots ``[B, new]`` of new tokens of the first ``B`` rows from ``positions [B]`` on, or of the rows of ``table``; where there is no page, -1, and
        ``lost`` is noted (:meth:`check`).  Without waiting for the device, in programs too."""
        rows, shared = positions.shape[0], 0 if table is not None else len(self._shared)
        table = self.page_table[:rows] if table is None else table
        held = torch.full((rows,), table.shape[1], dtype=torch.int32, device=table.device)
        return page_tables.assign(table, held, self._no_ring, self._no_span, positions, new, self.page_size, lens=lens,
                                  lengths=torch.full((rows,), -1, dtype=torch.long, device=table.device), shared=shared, short=self.lost, in_place=True).slots

    def reserve(self, row: int, tokens: int) -> None:
        """Room for a sequence of ``tokens`` tokens in all, the shared ones among them."""
        if tokens > self.max_seq_len:                             # the last page may hold more, the rotation tables end there
            raise ValueError(f"a sequence of {tokens} tokens is longer than max_seq_len {self.max_seq_len}")
        held = len(self._shared) + len(self._rows[row])
        pages = self._take(max(0, (tokens + self.page_size - 1) // self.page_size - held))
        if pages:
            self._rows[row] += pages
            self.page_table[row, held:held + len(pages)] = torch.tensor(pages, dtype=torch.int32, device=self.page_table.device)

    def reserve_rows(self, rows: int, tokens: int) -> None:
        """:meth:`reserve` for the first ``rows`` rows: all of them, or, where the pool has not as much, none."""
        want = max(0, (tokens + self.page_size - 1) // self.page_size - len(self._shared))
        need = sum(max(0, want - len(self._rows[r])) for r in range(rows))
        if tokens <= self.max_seq_len and need > len(self._free):
            raise RuntimeError(f"the key/value pool has {len(self._free)} pages left, {need} are needed")
        for r in range(rows):
            self.reserve(r, tokens)

    def cover(self, positions: torch.Tensor, tokens: int) -> None:
        """Room for ``tokens`` new tokens of every row from ``positions [B]`` on (negative: an idle row).  The positions are read on the host, which
        waits for them; inside :meth:`reserved_ahead`, and while a program is captured or recorded, nothing is looked at."""
        if self._ahead or self.in_program():
            return
        starts = positions.tolist()
        if any(0 <= first < self.shared_tokens for first in starts):            # its keys would be everybody's
            raise ValueError(f"positions {starts}: some lie inside the shared prefix of {self.shared_tokens} tokens, which rows do not write to")
        for row, first in enumerate(starts):
            if first >= 0:
                self.reserve(row, first + tokens)

    @contextmanager
    def reserved_ahead(self, rows: int, tokens: int) -> Iterator[None]:
        """:meth:`reserve_rows`, and the caller's word that no sequence gets longer than that inside: steps go on without waiting for positions."""
        self.reserve_rows(rows, tokens)
        before, self._ahead = self._ahead, True
        try:
            yield
        finally:
            self._ahead = before

    def release(self, row: int) -> None:
        """The row's own pages go back to the pool; the shared ones stay."""
        if self.in_program():
            raise RuntimeError("pages are given back on the host: not by a call that is captured or recorded")
        self.check()
        self._give_back(row)

    def _give_back(self, row: int) -> None:
        if self._rows[row]:
            self._free += self._rows[row][::-1]
            self._rows[row] = []
            self.page_table[row, len(self._shared):] = -1

    def take_shared(self, tokens: int) -> torch.Tensor:
        """Pages for a prefix of ``tokens`` tokens that every row begins with, in place of the one before → ``[n]`` int32 (who asked fills them).  All
        rows start anew.  Captured and recorded programs go on with another prefix of the same length; while there are any, another length is refused."""
        if tokens % self.page_size:
            raise ValueError(f"a shared prefix fills whole pages of {self.page_size} tokens, got {tokens}")
        if tokens > self.max_seq_len:
            raise ValueError(f"a prefix of {tokens} tokens is longer than max_seq_len {self.max_seq_len}")
        n = tokens // self.page_size
        if n > self.num_pages:
            raise RuntimeError(f"the key/value pool has {self.num_pages} pages, {n} are needed")
        if self.in_program():
            raise RuntimeError("a shared prefix cannot be taken by a call that is captured or recorded")
        if self._programs not in (None, n):
            raise RuntimeError(f"programs were captured or recorded behind a prefix of {self._programs * self.page_size} tokens and would go on with it, "
                               f"{tokens} are asked for: kv.forget_programs() when none of them is run any more")
        self.check()
        return self._share(n)

    def _share(self, n: int) -> torch.Tensor:
        for row in range(self.batch_size):
            self._give_back(row)
        self._free += self._shared[::-1]
        self._shared = self._take(n)
        self._shared_table[:] = -1
        pages = self._shared_table[:n]
        pages._plan_state = True
        pages.copy_(torch.tensor(self._shared, dtype=torch.int32, device=self.page_table.device))
        self.page_table[:] = -1
        self.page_table[:, :n] = pages
        self.shared_pages = pages if n else None
        return pages

    def drop_shared(self) -> None:
        """The shared pages go back to the pool, and all rows start anew: what should have filled them failed.  Programs that count on them have to wait
        for another prefix of their length."""
        self._share(0)

    def reset(self) -> None:
        """All pages go back to the pool, the shared ones too (:meth:`take_shared` of nothing)."""
        self.take_shared(0)


class DevicePagedKVCacheManager(PagedKVCacheManager):
    """Pages handed out on the device, by ``ops.page_tables.assign``: :meth:`slots` gives the rows of a step what pages they are short of, from positions
    that the host does not look at, in captured and recorded programs as outside.  A pool that runs short, and positions without a page, are noted in ``lost``
    and said by :meth:`check`, which the end of a sequence does not wait for; whoever calls a model's steps in a loop of their own calls it behind the last one, at the end of
    :meth:`reserved_ahead` it is called.  Rows of a prompt get pages for the tokens that count."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        device = self.page_table.device
        self.held = torch.zeros(self.batch_size, dtype=torch.int32, device=device)
        self.free = torch.arange(self.num_pages, dtype=torch.int32, device=device)
        self.span = torch.tensor([0, self.num_pages], device=device)
        self._row = torch.arange(self.batch_size, device=device)
        for t in (self.held, self.free, self.span):
            t._plan_state = True

    @property
    def free_pages(self) -> int:
        """Waits for the device."""
        taken, put = self.span.tolist()
        return put - taken

    def _assign(self, rows: int, positions: torch.Tensor, new: int = 0, lens=None, lengths=None) -> torch.Tensor:
        return page_tables.assign(self.page_table[:rows], self.held[:rows], self.free, self.span, positions, new, self.page_size, lens=lens, lengths=lengths,
                                  shared=len(self._shared), short=self.lost, in_place=True).slots

    def slots(self, positions, new, lens=None, table=None):
        """As in the class above, and pages for the tokens that have none."""
        return self._assign(positions.shape[0], positions, new, lens) if table is None else super().slots(positions, new, lens, table)

    def check(self) -> None:
        """Raises if tokens were left without a page since the last look, whose keys are missing from what came after: the pool was too small for its rows, or
        they are longer than ``max_seq_len``.  Waits for the device."""
        if bool(self.lost):
            self.lost.zero_()
            raise RuntimeError(f"tokens were left without a page, and their keys are lost: a pool of {self.num_pages} pages of {self.page_size} tokens ran short, or "
                               f"rows went on behind max_seq_len {self.max_seq_len}")

    def reserve(self, row: int, tokens: int) -> None:
        if tokens > self.max_seq_len:
            raise ValueError(f"a sequence of {tokens} tokens is longer than max_seq_len {self.max_seq_len}")
        if tokens > 0:
            self._assign(self.batch_size, self._row, lengths=torch.where(self._row == row, tokens, -1))

    def reserve_rows(self, rows: int, tokens: int) -> None:
        """:meth:`reserve` for the first ``rows`` rows, in their order, as far as the pool goes."""
        if tokens > self.max_seq_len:
            raise ValueError(f"a sequence of {tokens} tokens is longer than max_seq_len {self.max_seq_len}")
        if tokens > 0:
            self._assign(self.batch_size, self._row, lengths=torch.where(self._row < rows, tokens, -1))

    def cover(self, positions: torch.Tensor, tokens: int) -> None:
        """:meth:`slots` does that."""

    @contextmanager
    def reserved_ahead(self, rows: int, tokens: int) -> Iterator[None]:
        """Rows get their pages when they need them, and nothing ahead: what had no page is said at the end (:meth:`check`, which waits for the device; what was lost
        before, at the beginning)."""
        if tokens > self.max_seq_len:
            raise ValueError(f"a sequence of {tokens} tokens is longer than max_seq_len {self.max_seq_len}")
        if not self.in_program():
            self.check()
        yield
        if not self.in_program():
            self.check()

    def release(self, row: int) -> None:
        self._assign(self.batch_size, self._row, lengths=torch.where(self._row == row, 0, -1))

    def _share(self, n: int) -> torch.Tensor:
        # all rows start anew: the first pages of the pool are everybody's, the others free
        self._shared = list(range(n))
        self._shared_table[:] = -1
        pages = self._shared_table[:n]
        pages._plan_state = True
        pages.copy_(torch.arange(n, dtype=torch.int32, device=pages.device))
        self.page_table[:] = -1
        self.page_table[:, :n] = pages
        self.held.fill_(n)
        self.free.copy_(torch.arange(self.num_pages, dtype=torch.int32, device=pages.device).roll(-n))
        self.span.copy_(torch.tensor([0, self.num_pages - n], device=pages.device))
        self.shared_pages = pages if n else None
        return pages
