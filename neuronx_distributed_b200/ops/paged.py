"""A key/value cache in pages: appending new tokens with the position rotation on the way, and attention over the pages
(kernels: ``csrc/paged.cu``).  What the reference keeps in contiguous rows per sequence (``examples/inference/modules/kvcache/
kv_cache_manager.py:60-199``) lies here in pages of one pool, so that sequences of unequal length, and ones that begin alike, share it.

Layout: caches ``[pages, page_size, Hkv, D]`` (any strides with contiguous ``D``; a multiple of 16 tokens a page), ``page_table [B, n]`` int32: the
page of tokens ``i * page_size …`` of a sequence.  New tokens ``[B, W, heads, D]``; row ``b``'s stand at ``positions[b] … positions[b] + W - 1``, of
which the first ``lens[b]`` count (``None``: all).  A negative position is an idle row of the batch.  Entries of the table outside the pool are holes:
nothing is written there and nobody sees their keys.  Two rows that append to the same place of the same page leave either's numbers.

Serving only: there is no gradient, and tensors that ask for one are refused.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ext


def _ints(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _table(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and (t.dim() != 2 or t.shape[1] <= 1 or t.stride(1) == 1) else t.to(torch.int32).contiguous()


def _no_gradient(name: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or with tensors that ask for none")


def _kernels(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ok: str):
    """The extension, whose entry points take what is for their kernels and return None for the rest; a recorded call has to be one that they take."""
    if not _ext.use_cuda(q):
        return None
    if _ext._PLAN_PROXY is not None and not getattr(_ext._load(), ok)(q, k_cache, v_cache):
        return None
    return _ext.ext()


def _check(q, k_cache, v_cache, page_table, positions, lens) -> None:
    """The refusals of ``csrc/paged_binding.cpp`` for tensors that the kernels do not take."""
    def need(ok, text):
        if not ok:
            raise ValueError(text)

    need(q.dim() == 4 and k_cache.dim() == 4 and v_cache.dim() == 4,
         "queries are [batch, new tokens, heads, head size], caches [pages, page size, heads, head size]")
    need(k_cache.shape == v_cache.shape and k_cache.shape[3] == q.shape[3] and k_cache.shape[2] > 0 and q.shape[2] > 0
         and q.shape[2] % k_cache.shape[2] == 0,
         f"heads do not match: queries {tuple(q.shape)}, keys {tuple(k_cache.shape)}, values {tuple(v_cache.shape)}")
    need(q.dtype == k_cache.dtype == v_cache.dtype, "queries and caches are of one type")
    need(all(t.device == q.device for t in (k_cache, v_cache, page_table, positions)), "all tensors are on one device")
    need(k_cache.shape[0] > 0 and k_cache.shape[1] > 0 and k_cache.shape[1] % 16 == 0, f"a page holds a multiple of 16 tokens, got {k_cache.shape[1]}")
    need(page_table.dim() == 2 and page_table.shape[0] == q.shape[0], f"page_table must be [{q.shape[0]}, pages of a sequence], got {tuple(page_table.shape)}")
    need(positions.dim() == 1 and positions.shape[0] == q.shape[0], f"positions must be [{q.shape[0]}], got {tuple(positions.shape)}")
    need(lens is None or (lens.dim() == 1 and lens.shape[0] == q.shape[0] and lens.device == q.device), f"lens must be [{q.shape[0]}] on {q.device}")


def _new_tokens(positions, lens, W: int) -> torch.Tensor:
    """How many of a row's tokens count, ``[B]``."""
    n = torch.full_like(positions, W) if lens is None else lens.clamp(0, W)
    return torch.where(positions < 0, torch.zeros_like(n), n)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lens: Optional[torch.Tensor] = None,
                lost: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates ``q [B, W, H, D]`` (returned, ``[W, B, H, D]`` in memory) and ``k [B, W, Hkv, D]`` by their tokens' positions, and writes ``k`` and ``v``
    to the pages, in one launch.  ``cos`` / ``sin [positions, D / 2]`` fp32: :func:`ops.rope.rope_tables`.  Tokens that do not count, or that stand
    behind the tables' end, come back as zeros and are not written; tokens behind the page table's end are not written.  ``lost [1]`` int32 becomes 1
    where a token that counts was not written (and stays as it is otherwise)."""
    _no_gradient("rope_append", q, k, v, k_cache, v_cache)
    e = _kernels(q, k_cache, v_cache, "paged_append_ok")
    if e is not None:
        out = e.paged_append(q, k, v, positions, cos, sin, k_cache, v_cache, page_table, lens, lost)
        if out is not None:
            return out
    positions, page_table = _ints(positions, torch.long).clamp(-1, 1 << 40), _table(page_table)
    lens = None if lens is None else _ints(lens, torch.long)
    _check(q, k_cache, v_cache, page_table, positions, lens)
    if lost is not None and (lost.dtype != torch.int32 or lost.shape != (1,) or lost.device != q.device):
        raise ValueError("lost must be an int32 tensor of one number on the queries' device")
    B, W, H, D = q.shape
    if k.shape != v.shape or tuple(k.shape) != (B, W, k_cache.shape[2], D):
        raise ValueError(f"new keys and values must be [{B}, {W}, {k_cache.shape[2]}, {D}]")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("queries, keys and values are of one type and on one device")
    if (cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] * 2 != D or cos.dtype != torch.float32 or sin.dtype != torch.float32
            or cos.device != q.device or sin.device != q.device):
        raise ValueError(f"cos and sin must be contiguous float32 tables [positions, {D // 2}]")
    w = torch.arange(W, device=q.device)
    p = positions[:, None] + w
    counts = w < _new_tokens(positions, lens, W)[:, None]
    live = counts & (p < cos.shape[0])
    at = p.clamp(0, max(cos.shape[0] - 1, 0))
    c, s = cos[at][:, :, None], sin[at][:, :, None]

    def rotate(x):
        a, b = x[..., :D // 2].float(), x[..., D // 2:].float()
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    ps = k_cache.shape[1]
    column = p // ps
    held = live & (column < page_table.shape[1])
    page = page_table.long().gather(1, column.clamp(0, max(page_table.shape[1] - 1, 0))) if page_table.shape[1] else torch.full_like(p, -1)
    held &= (page >= 0) & (page < k_cache.shape[0])
    if lost is not None:
        lost.logical_or_((counts & ~held).any())
    k_cache[page[held], (p % ps)[held]] = rotate(k).to(k_cache.dtype)[held]
    v_cache[page[held], (p % ps)[held]] = v[held]
    return rotate(q).masked_fill(~live[:, :, None, None], 0.0).to(q.dtype).transpose(0, 1).contiguous().transpose(0, 1)


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor,
              scale: Optional[float] = None, lens: Optional[torch.Tensor] = None, shared_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens ``q [B, W, H, D]`` (their keys are in the pages already) over the cache → ``[B, W, H, D]`` (``[W, B, H, D]`` in
    memory): token ``w`` of row ``b`` sees keys ``0 … positions[b] + w``.  ``W`` = 1: token generation; a few: a drafted window; many: a portion
    of a prompt.  Tokens that do not count, or see no key, come back as zeros.  Keys and values that some token of a row sees have to be finite, and
    scores, held in 32 bits, below 2^30 in magnitude.

    Sums and statistics are in 32 bits.  Weights are rounded to the cache's type before they meet the values where a sequence has more than 16 query rows
    for a key/value head (tokens times heads of a group; more than 8 of long sequences), and over pages that all share where the batch has; fewer rows
    keep them.  The sizes of tables, not positions, say which kernel it is: one sequence in a table for many tokens takes longer than in a narrow one.

    ``shared_pages [n]`` int32: the pages of the first ``n * page_size`` tokens of EVERY sequence; the first ``n`` columns of ``page_table`` are not
    looked at.  Where a sequence has up to 128 query rows (tokens times heads of a group), they are read once for the whole batch."""
    _no_gradient("paged attention", q, k_cache, v_cache)
    e = _kernels(q, k_cache, v_cache, "paged_attention_ok")
    if e is not None:
        out = e.paged_attention(q, k_cache, v_cache, page_table, positions, scale, lens, shared_pages)
        if out is not None:
            return out
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    positions, page_table = _ints(positions, torch.long).clamp(-1, 1 << 40), _table(page_table)
    lens = None if lens is None else _ints(lens, torch.long)
    if shared_pages is not None:
        shared_pages = _ints(shared_pages, torch.int32)
    _check(q, k_cache, v_cache, page_table, positions, lens)
    if not 0 < scale < 1e30:
        raise ValueError("the scale of the scores is positive")
    if shared_pages is not None:
        if shared_pages.dim() != 1 or shared_pages.device != q.device or shared_pages.shape[0] > page_table.shape[1]:
            raise ValueError("shared_pages is a list of no more pages than page_table has, on the queries' device")
        page_table = torch.cat([shared_pages.expand(q.shape[0], -1), page_table[:, shared_pages.shape[0]:]], 1)
    return _attention_plain(q, k_cache, v_cache, page_table, positions, scale, lens)


def _attention_plain(q, k_cache, v_cache, page_table, positions, scale, lens):
    B, W, H, D = q.shape
    pages, ps, Hkv, _ = k_cache.shape
    if q.numel() == 0 or page_table.shape[1] == 0:
        return torch.zeros_like(q)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    there = (page_table >= 0) & (page_table < pages)
    at = page_table.long().clamp(0, pages - 1)
    keys = torch.arange(page_table.shape[1] * ps, device=q.device)
    new = _new_tokens(positions, lens, W)
    w = torch.arange(W, device=q.device)
    end = positions + new                                     # [B] keys that anybody of the row sees
    held = there.repeat_interleave(ps, 1) & (keys < end[:, None])
    # numbers that nobody sees may be anything
    k = k_cache[at].flatten(1, 2).to(wide).masked_fill(~held[:, :, None, None], 0.0).transpose(1, 2)
    v = v_cache[at].flatten(1, 2).to(wide).masked_fill(~held[:, :, None, None], 0.0).transpose(1, 2)
    seen = held[:, None] & (keys <= (positions[:, None] + w)[..., None]) & (w < new[:, None])[..., None]      # [B, W, keys]
    G = H // Hkv
    s = q.to(wide).view(B, W, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, W * G, D) @ k.transpose(2, 3) * scale
    s = s.masked_fill(~seen.repeat_interleave(G, 1)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / total.masked_fill(total == 0, 1.0)
    return o.view(B, Hkv, W, G, D).permute(2, 0, 1, 3, 4).reshape(W, B, H, D).to(q.dtype).transpose(0, 1)
