"""A key/value cache in pages that is held in 4 bits: appending new tokens with the position rotation on the way, reading tokens back, and attention over
the codes (kernels: ``csrc/paged_int4.cu``).  What ``ops.paged`` does for 16-bit pages, in 5 bits a number; the reference keeps 8-bit rows at the least
(``examples/inference/modules/kvcache/kv_cache_manager.py:60-199``).

Format: 32 numbers ``x`` of a token's head, one after the other, are held as ``m + s c``: ``m`` is their least and ``s`` a fifteenth of what the largest
is above ``m``, both rounded to half precision, and ``c`` is ``(x - m) / s`` rounded to the nearest of 0 … 15 (0 where ``s`` is 0 or not finite).  A number
is off by ``s / 2`` at most, and by what the roundings of ``m`` and ``s`` do at the ends.  A least number beyond half precision, or a range of 15 times that, makes its 32 infinite
or NaN; a largest one that is does not by itself.

Layout (:class:`Pages`): ``codes [pages, page_size, Hkv, D / 2]`` uint8, number ``2 i`` of a head in the low half of byte ``i``; ``steps [pages, page_size,
Hkv, 2, D / 32]`` float16, first ``s``, then ``m``.  A page has a multiple of 16 tokens.  :func:`new_pages` lays a head's rows of a page beside one another.
New tokens ``[B, W, heads, D]``; where they go is said by slots ``[B, W]`` int32, ``page * page_size + place``, -1: nowhere (``ops.page_tables.assign``).

Serving only: there is no gradient, and tensors that ask for one are refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _ext
from .paged import _attention_plain, _ints, _no_gradient, _table

GROUP = 32


class Pages(NamedTuple):
    """Keys or values of a pool of pages."""
    codes: torch.Tensor
    steps: torch.Tensor


def new_pages(pages: int, page_size: int, heads: int, dim: int, device=None) -> Pages:
    """A pool of zeros."""
    if page_size < 16 or page_size % 16:
        raise ValueError(f"a page holds a multiple of 16 tokens, got {page_size}")
    if dim <= 0 or dim % GROUP:
        raise ValueError(f"heads of a multiple of {GROUP} numbers are held in 4 bits, got {dim}")
    if pages < 1 or heads < 1:
        raise ValueError("a pool without pages or heads")
    return Pages(torch.zeros(pages, heads, page_size, dim // 2, dtype=torch.uint8, device=device).transpose(1, 2),
                 torch.zeros(pages, heads, page_size, 2, dim // GROUP, dtype=torch.float16, device=device).transpose(1, 2))


def pack(x: torch.Tensor) -> Pages:
    """Codes ``[..., D / 2]`` and steps ``[..., 2, D / 32]`` of numbers ``[..., D]``, from 64 bits."""
    if x.shape[-1] % GROUP:
        raise ValueError(f"heads of a multiple of {GROUP} numbers are held in 4 bits, got {x.shape[-1]}")
    x = x.double().unflatten(-1, (-1, GROUP))
    lo = x.amin(-1).half()
    step = ((x.amax(-1) - lo.double()) / 15).half()
    c = ((x - lo.double()[..., None]) / step.double()[..., None]).round().clamp(0, 15)
    c = torch.where(((step > 0) & step.isfinite())[..., None], c, 0.0).to(torch.uint8).flatten(-2)
    return Pages(c[..., ::2] | c[..., 1::2] << 4, torch.stack([step, lo], -2))


def unpack(pages: Pages, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """What codes ``[..., D / 2]`` and steps ``[..., 2, D / 32]`` stand for, ``[..., D]``."""
    c = torch.stack([pages.codes & 15, pages.codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP))
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    return (c.to(wide) * pages.steps[..., 0, :, None].to(wide) + pages.steps[..., 1, :, None].to(wide)).flatten(-2).to(dtype)


def _check_pages(k: Pages, v: Pages, heads: Optional[int] = None, dim: Optional[int] = None, device=None) -> None:
    """The refusals of ``csrc/paged_int4_binding.cpp``."""
    def need(ok, text):
        if not ok:
            raise ValueError(text)

    for p in (k, v):
        need(p.codes.dim() == 4 and p.codes.dtype == torch.uint8 and p.steps.dim() == 5 and p.steps.dtype == torch.float16,
             "pages are uint8 codes [pages, page size, heads, head size / 2] and float16 steps [pages, page size, heads, 2, head size / 32]")
        need(p.codes.shape[:3] == p.steps.shape[:3] and p.codes.shape[3] > 0 and p.codes.shape[3] % 16 == 0 and p.steps.shape[3] == 2
             and p.steps.shape[4] * 16 == p.codes.shape[3], f"codes {tuple(p.codes.shape)} and steps {tuple(p.steps.shape)} do not match")
    need(k.codes.shape == v.codes.shape, f"keys {tuple(k.codes.shape)} and values {tuple(v.codes.shape)} do not match")
    need(all(t.device == k.codes.device for t in (*k, *v)) and (device is None or k.codes.device == device), "all tensors are on one device")
    pages, ps, Hkv, half = k.codes.shape
    need(pages > 0 and Hkv > 0 and ps > 0 and ps % 16 == 0, f"a page holds a multiple of 16 tokens, got {ps}")
    need(pages * ps < 1 << 31, "a pool of too many tokens")
    need(heads is None or heads > 0 and heads % Hkv == 0, f"{heads} query heads do not go with {Hkv} key heads")
    need(dim is None or dim == 2 * half, f"heads of {dim} numbers, pages of {2 * half}")


def _kernels(first: torch.Tensor, ok: str, *args):
    """The extension, whose entry points take what is for their kernels and return None for the rest; a recorded call has to be one that they take.  (Callers go by
    the extension itself where nothing is recorded: 0.4 us of a call's six.)"""
    if not _ext.use_cuda(first) or (_ext._PLAN_PROXY is not None and not getattr(_ext._load(), ok)(*args)):
        return None
    return _ext.ext()


def _check_slots(slots, B: int, W: int, device) -> torch.Tensor:
    if slots.shape != (B, W) or slots.device != device or slots.dtype.is_floating_point:
        raise ValueError(f"slots must be whole numbers [{B}, {W}] on {device}")
    return _ints(slots, torch.long)


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: Pages, v_pages: Pages,
           slots: torch.Tensor, interleaved: bool = False, lost: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates ``q [B, W, H, D]`` (returned, ``[W, B, H, D]`` in memory) and ``k [B, W, Hkv, D]`` by their tokens' positions ``positions[b] + w``, and writes
    the codes of ``k`` and ``v`` to the tokens' slots, in one launch.  ``cos`` / ``sin [positions, r / 2]`` fp32 (``ops.rope.rope_tables``): the first ``r``
    numbers of a head turn, number ``i`` with ``i + r / 2``, or with ``interleaved`` number ``2 i`` with ``2 i + 1``; the others stay.  Tokens without a
    slot, or that stand outside the rotation tables, come back as zeros and are not written.  ``lost [1]`` int32 becomes 1 where a token that has a slot
    stands outside the tables (and stays as it is otherwise).  What a slot holds that two tokens of a call have is not defined.

    Codes are those of the rotated numbers before any rounding: next to a border they are found in 64 bits."""
    _no_gradient("append", q, k, v)
    e = _ext._load() if _ext._PLAN_PROXY is None and _ext.use_cuda(q) else _kernels(q, "int4_append_ok", q, *k_pages, *v_pages, cos, interleaved)
    if e is not None:
        out = e.int4_append(q, k, v, positions, cos, sin, *k_pages, *v_pages, slots, interleaved, lost)
        if out is not None:
            return out
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError("queries are [batch, new tokens, heads, head size], new keys and values [batch, new tokens, key heads, head size]")
    B, W, H, D = q.shape
    _check_pages(k_pages, v_pages, H, D, q.device)
    if k.shape[2] != k_pages.codes.shape[2]:
        raise ValueError(f"new keys and values must be [{B}, {W}, {k_pages.codes.shape[2]}, {D}]")
    if not q.dtype.is_floating_point or k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("queries, keys and values are of one type and on one device")
    if (cos.dim() != 2 or cos.shape != sin.shape or not 0 <= cos.shape[1] * 2 <= D or cos.dtype != torch.float32 or sin.dtype != torch.float32
            or cos.device != q.device or sin.device != q.device):
        raise ValueError(f"cos and sin must be float32 tables [positions, at most {D // 2}] on the queries' device")
    if positions.shape != (B,) or positions.device != q.device:
        raise ValueError(f"positions must be [{B}] on {q.device}")
    if lost is not None and (lost.dtype != torch.int32 or lost.shape != (1,) or lost.device != q.device):
        raise ValueError("lost must be an int32 tensor of one number on the queries' device")
    slots = _check_slots(slots, B, W, q.device)
    half, ps = cos.shape[1], k_pages.codes.shape[1]
    p = _ints(positions, torch.long).clamp(-1 << 40, 1 << 40)[:, None] + torch.arange(W, device=q.device)
    has = (slots >= 0) & (slots < k_pages.codes.shape[0] * ps)
    live = has & (p >= 0) & (p < cos.shape[0])
    if lost is not None:
        lost.logical_or_((has & ~live).any())
    at = p.clamp(0, max(cos.shape[0] - 1, 0))
    c, s = (t[at][:, :, None].double() if t.shape[0] else t.new_zeros(B, W, 1, half).double() for t in (cos, sin))

    def rotate(x):
        t, rest = x[..., :2 * half].double(), x[..., 2 * half:].double()
        a, b = (t[..., ::2], t[..., 1::2]) if interleaved else (t[..., :half], t[..., half:])
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1 if interleaved else -2).flatten(-2), rest], -1)

    where = slots[live]
    for x, pages in ((rotate(k), k_pages), (v, v_pages)):
        for dst, src in zip(pages, pack(x[live])):
            dst[where // ps, where % ps] = src
    return rotate(q).masked_fill(~live[:, :, None, None], 0.0).to(q.dtype).transpose(0, 1).contiguous().transpose(0, 1)


def gather(k_pages: Pages, v_pages: Pages, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of the tokens at ``slots [B, W]``, ``[B, W, Hkv, D]`` each, zeros where there is no slot, in one launch."""
    e = _ext._load() if _ext._PLAN_PROXY is None and _ext.use_cuda(k_pages.codes) else _kernels(k_pages.codes, "int4_gather_ok", *k_pages, *v_pages, dtype)
    if e is not None:
        out = e.int4_gather(*k_pages, *v_pages, slots, dtype)
        if out is not None:
            return tuple(out)
    if slots.dim() != 2 or not dtype.is_floating_point:
        raise ValueError("slots are [batch, tokens], and numbers are read as floating-point ones")
    _check_pages(k_pages, v_pages, device=slots.device)
    slots = _check_slots(slots, *slots.shape, k_pages.codes.device)
    pages, ps = k_pages.codes.shape[:2]
    live = (slots >= 0) & (slots < pages * ps)
    at = slots.clamp(0, pages * ps - 1)
    return tuple(unpack(Pages(p.codes[at // ps, at % ps], p.steps[at // ps, at % ps]), dtype).masked_fill(~live[:, :, None, None], 0.0)
                 for p in (k_pages, v_pages))


def attention(q: torch.Tensor, k_pages: Pages, v_pages: Pages, page_table: torch.Tensor, positions: torch.Tensor, scale: Optional[float] = None,
              lens: Optional[torch.Tensor] = None, shared_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens ``q [B, W, H, D]`` over a cache in 4 bits → ``[B, W, H, D]`` (``[W, B, H, D]`` in memory): as ``ops.paged.attention``
    of the numbers that the codes stand for, with its arguments.  ``page_table [B, n]`` int32 (entries outside the pool are holes, whose keys nobody
    sees), ``positions [B]`` of the rows' first new tokens (negative: an idle row), ``lens [B]`` new tokens that count.  ``shared_pages [n]`` int32 stand in
    place of the first ``n`` columns of every row's table; each row reads them for itself.  Keys and values that some token of a row sees have to be
    131008 at most in magnitude (twice the largest half), queries finite and below 1e35.  The kernels take pools whose codes span less than 64 GB, and tables of less than 2^31 tokens.

    Scaled scores stay below 2^24 in magnitude.  Sums and statistics are in 32 bits.  Where a sequence has up to 8 query rows for a key/value head (tokens times heads of a
    group), codes and steps enter as they are; weights, and their products with the steps of the values, are rounded to halves, to two halves each where the result is in half
    precision.  With more rows values are rounded to halves before they meet such weights; and portions of prompts in bf16 read pages that were unpacked to halves before, keys as
    well, and weights of one half: the error of a score is that of its keys.  The sizes of tables, not positions, say which kernel it is."""
    _no_gradient("attention in 4 bits", q)
    e = _ext._load() if _ext._PLAN_PROXY is None and _ext.use_cuda(q) else _kernels(q, "int4_attention_ok", q, *k_pages, *v_pages)
    if e is not None:
        out = e.int4_attention(q, *k_pages, *v_pages, page_table, positions, scale, lens, shared_pages)
        if out is not None:
            return out
    if q.dim() != 4 or not q.dtype.is_floating_point:
        raise ValueError("queries are floating-point numbers [batch, new tokens, heads, head size]")
    B, W, H, D = q.shape
    _check_pages(k_pages, v_pages, H, D, q.device)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0 < scale < 1e30:
        raise ValueError("the scale of the scores is positive")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.device != q.device:
        raise ValueError(f"page_table must be [{B}, pages of a sequence] on {q.device}")
    if positions.shape != (B,) or positions.device != q.device:
        raise ValueError(f"positions must be [{B}] on {q.device}")
    if lens is not None and (lens.shape != (B,) or lens.device != q.device):
        raise ValueError(f"lens must be [{B}] on {q.device}")
    page_table = _table(page_table)
    if shared_pages is not None:
        if shared_pages.dim() != 1 or shared_pages.device != q.device or shared_pages.shape[0] > page_table.shape[1]:
            raise ValueError("shared_pages is a list of no more pages than page_table has, on the queries' device")
        page_table = torch.cat([_ints(shared_pages, torch.int32).expand(B, -1), page_table[:, shared_pages.shape[0]:]], 1)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    used = page_table.long().clamp(0, k_pages.codes.shape[0] - 1).flatten()         # only what the table names is unpacked
    k, v = (unpack(Pages(p.codes[used], p.steps[used]), wide) for p in (k_pages, v_pages))
    there = (page_table >= 0) & (page_table < k_pages.codes.shape[0])
    table = torch.where(there, torch.arange(page_table.numel(), device=q.device, dtype=torch.int32).view(page_table.shape), -1)
    if not used.numel():
        return torch.zeros(W, B, H, D, dtype=q.dtype, device=q.device).transpose(0, 1)
    out = _attention_plain(q.to(wide), k, v, table, _ints(positions, torch.long).clamp(-1, 1 << 40), scale, None if lens is None else _ints(lens, torch.long))
    return out.to(q.dtype).transpose(0, 1).contiguous().transpose(0, 1)
