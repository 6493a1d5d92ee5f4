"""Page tables of a batch and the slots of its new tokens, from the lengths of its requests, on the device (kernel: ``csrc/page_tables.cu``).
Nothing waits for the host, so a captured program can take pages.  The reference's cache has a row per sequence and needs no tables
(``examples/inference/modules/kvcache/kv_cache_manager.py:60-199``).

State: ``page_table [B, n]`` int32 (a row's pages in the order of its tokens), ``held [B]`` int32 (columns of a row that have a page; the first ``shared``
columns are everybody's and never change), and the free pages: a ring ``free [P]`` int32, ``P`` the pages of the pool, with ``span [2]`` int64: the count
of pages that were ever taken from it and that were ever put into it (place ``i`` of either is ``free[i % P]``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _ext
from .paged import _ints


class Tables(NamedTuple):
    page_table: torch.Tensor
    held: torch.Tensor
    free: torch.Tensor
    span: torch.Tensor
    slots: torch.Tensor


def assign(page_table: torch.Tensor, held: torch.Tensor, free: torch.Tensor, span: torch.Tensor, positions: torch.Tensor, new: int, page_size: int,
           lens: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, shared: int = 0, trim: bool = False,
           short: Optional[torch.Tensor] = None, in_place: bool = False) -> Tables:
    """Pages for all rows, and ``slots [B, new]`` int32 of their new tokens: ``page * page_size + place``, in one launch.

    Row ``b``'s new tokens stand at ``positions[b] … positions[b] + new - 1``, of which the first ``lens[b]`` count (``None``: all; a negative position:
    none).  ``lengths[b]``: the tokens that the row has to have room for; 0: it ends, its own pages go back; negative: it stays as it is.  ``None``: up
    to its new tokens, and rows without any stay.  ``trim``: pages behind ``lengths`` go back too; otherwise rows keep them.

    Pages are taken in the order of the rows, from the ring as it was before the call; the first row that finds too few, and the rows behind it, take
    none.  A row that would need more columns than the table has takes none.  Tokens that do not count, that stand in the shared columns, or for which
    there is no page, have slot -1.  ``short [1]`` int32 becomes 1 where a row that needed pages took none, or a token that counts has no slot (and stays
    as it is otherwise).

    ``in_place``: the state's own tensors are changed and returned (rows of the table may not share memory, and calls that change one state go one after the
    other); otherwise they stay, and new ones are returned."""
    if _ext.use_cuda(page_table):
        return Tables(*_ext.ext().assign_pages(page_table, held, free, span, positions, new, page_size, lens, lengths, shared, trim, short, in_place))
    return _assign_plain(page_table, held, free, span, positions, new, page_size, lens, lengths, shared, trim, short, in_place)


def _check(page_table, held, free, span, positions, new, page_size, lens, lengths, shared, short, in_place) -> None:
    """The refusals of ``csrc/paged_int4_binding.cpp``."""
    def need(ok, text):
        if not ok:
            raise ValueError(text)

    dev = page_table.device
    need(page_table.dim() == 2 and page_table.dtype == torch.int32 and (page_table.shape[1] <= 1 or page_table.stride(1) == 1),
         "page_table must be an int32 tensor [batch, pages of a sequence]")
    B, n = page_table.shape
    for t, name, dtype, size in ((held, "held", torch.int32, B), (span, "span", torch.int64, 2)):
        need(t.dtype == dtype and t.shape == (size,) and t.is_contiguous() and t.device == dev,
             f"{name} must be a contiguous {dtype} tensor of {size} numbers on the tables' device")
    need(free.dtype == torch.int32 and free.dim() == 1 and free.shape[0] > 0 and free.is_contiguous() and free.device == dev,
         "free must be a contiguous int32 tensor with a place for every page of the pool")
    for t, name in ((positions, "positions"), (lens, "lens"), (lengths, "lengths")):
        need(t is None and name != "positions" or t is not None and t.shape == (B,) and t.device == dev, f"{name} must be [{B}] on the tables' device")
    need(new >= 0 and page_size > 0 and free.shape[0] * page_size < 1 << 31 and n < 1 << 30 and n * page_size < 1 << 31 and B * max(new, 1) < 1 << 31 and B < 1 << 15,
         f"too many tokens: {free.shape[0]} pages of {page_size}, {B} rows of {new} new tokens")
    need(not in_place or B <= 1 or page_table.stride(0) >= n, "rows of a page_table that is changed in place lie apart")
    need(0 <= shared <= n, f"shared columns: {shared} of {n}")
    need(short is None or (short.dtype == torch.int32 and short.shape == (1,) and short.device == dev),
         "short must be an int32 tensor of one number on the tables' device")


def _assign_plain(page_table, held, free, span, positions, new, page_size, lens, lengths, shared, trim, short, in_place) -> Tables:
    _check(page_table, held, free, span, positions, new, page_size, lens, lengths, shared, short, in_place)
    (B, n), P, dev = page_table.shape, free.shape[0], page_table.device
    positions = _ints(positions, torch.long).clamp(-1, 1 << 40)
    counts = torch.full_like(positions, new) if lens is None else _ints(lens, torch.long).clamp(0, new)
    counts = torch.where(positions < 0, 0, counts)
    lengths = torch.where(counts > 0, positions + counts, -1) if lengths is None else _ints(lengths, torch.long).clamp(-1, 1 << 40)
    had = held.long().clamp(shared, n)
    want = torch.where(lengths > 0, (lengths + page_size - 1) // page_size, 0)
    take = torch.where(want <= n, (want - had).clamp(min=0), 0)
    upto = take.cumsum(0)
    fits = upto <= span[1] - span[0]
    few = (want > n).any() | ((take > 0) & ~fits).any()
    take = torch.where(fits, take, 0)
    ends = (lengths >= 0) if trim else (lengths == 0)
    give = torch.where(ends, (had - want.clamp(min=shared)).clamp(min=0), 0)
    back = give.cumsum(0) - give
    column = torch.arange(n, device=dev)
    taken = (column >= had[:, None]) & (column < (had + take)[:, None])
    given = (column >= (had - give)[:, None]) & (column < had[:, None])
    fresh = free[(span[0] + (upto - take)[:, None] + column - had[:, None]) % P]
    table = torch.where(taken, fresh, torch.where(given, -1, page_table))
    ring = free.clone()
    places = (span[1] + back[:, None] + column - (had - give)[:, None]) % P
    ring[places[given]] = page_table[given]
    p = positions[:, None] + torch.arange(new, device=dev)
    column = p // page_size
    counted = torch.arange(new, device=dev) < counts[:, None]
    there = counted & (column >= shared) & (column < (had + take - give)[:, None])
    page = table.long().gather(1, column.clamp(0, max(n - 1, 0))) if n else torch.full_like(p, -1)
    there &= (page >= 0) & (page < P)
    slots = torch.where(there, page * page_size + p % page_size, -1).int()
    if short is not None:
        short.logical_or_(few | (counted & ~there).any())
    out = (table, (had + take - give).int(), ring, span + torch.stack([take.sum(), give.sum()]))
    if in_place:
        for t, now in zip((page_table, held, free, span), out):
            t.copy_(now)
        out = (page_table, held, free, span)
    return Tables(*out, slots)
