"""Key/value cache in pages: one pool per layer ``[pages, page_size, H_kv_local, D]``, a table of pages per batch row, and a prefix that all rows
share.  Beside ``kv_cache.py``, whose rows are contiguous and as long as the longest sequence may get, rows here hold as many pages as they need,
and what they begin alike is there once.  The pages themselves are written and read by ``ops.paged`` (``csrc/paged.cu``); this class says
whose they are.  Tables live on the device at fixed addresses (captured and recorded programs read them as they are when they run); pages are handed
out on the host, so a program takes none: its rows have to be reserved before it runs (:meth:`PagedKVCacheManager.check` says whether they were), and
the length of the shared prefix is part of it."""
from __future__ import annotations

from contextlib import contextmanager
from typing import Iterator, List, Optional

import torch

from ..utils.plan_registry import recording


class PagedKVCacheManager:
    def __init__(self, num_layers: int, batch_size: int, max_seq_len: int, num_kv_heads_local: int, head_dim: int, page_size: int = 32,
                 num_pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device=None):
        """``num_pages``: of the pool (default: enough for every row to be ``max_seq_len`` long)."""
        if page_size < 16 or page_size % 16:
            raise ValueError(f"a page holds a multiple of 16 tokens, got {page_size}")
        self.num_layers, self.batch_size, self.max_seq_len, self.page_size = num_layers, batch_size, max_seq_len, page_size
        self.columns = (max_seq_len + page_size - 1) // page_size
        self.num_pages = batch_size * self.columns if num_pages is None else num_pages
        if self.num_pages < 1:
            raise ValueError("a pool without pages")
        shape = (self.num_pages, page_size, num_kv_heads_local, head_dim)
        self.k: List[torch.Tensor] = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v: List[torch.Tensor] = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.page_table = torch.full((batch_size, self.columns), -1, dtype=torch.int32, device=device)
        self._shared_table = torch.full((self.columns,), -1, dtype=torch.int32, device=device)
        self.shared_pages: Optional[torch.Tensor] = None      # [n] int32, the beginning of that table: what every row begins with
        self.page_table._plan_state = True                    # a launch plan keeps nothing that follows from it (inference/launch_plan.py)
        self.lost = torch.zeros(1, dtype=torch.int32, device=device)        # becomes 1 where a token had no page (ops.paged.rope_append)
        self._shared: List[int] = []
        self._rows: List[List[int]] = [[] for _ in range(batch_size)]       # pages of a row behind the shared ones
        self._free: List[int] = list(range(self.num_pages))[::-1]
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
