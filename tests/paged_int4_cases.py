"""Oracles and random inputs of the paged cache in 4 bits and of page tables: from their definitions, in 64 bits, one row at a time."""
import torch

import paged_cases
import paged_oracle

from neuronx_distributed_b200.ops.paged_int4 import Pages


def values(pages):
    """What codes and steps stand for."""
    c, s = pages.codes, pages.steps.double()
    D = c.shape[-1] * 2
    x = torch.empty(*c.shape[:-1], D, dtype=torch.float64, device=c.device)
    x[..., 0::2], x[..., 1::2] = (c % 16).double(), (c // 16).double()
    at = torch.arange(D, device=c.device) // 32
    return s[..., 1, :][..., at] + s[..., 0, :][..., at] * x


def sizes(pages):
    """Magnitudes of the two terms of a number."""
    return values(Pages(pages.codes, pages.steps.abs()))


def packed(x):
    """Codes and steps of ``x [..., D]``, a group of 32 at a time."""
    x = x.double()
    D = x.shape[-1]
    codes = torch.zeros(*x.shape[:-1], D // 2, dtype=torch.uint8, device=x.device)
    steps = torch.zeros(*x.shape[:-1], 2, D // 32, dtype=torch.float16, device=x.device)
    for g in range(D // 32):
        part = x[..., 32 * g:32 * g + 32]
        m = part.min(-1).values.half()
        s = ((part.max(-1).values - m.double()) / 15).half()
        ok = (s > 0) & s.isfinite()
        c = torch.where(ok[..., None], torch.round((part - m.double()[..., None]) / torch.where(ok, s, 1).double()[..., None]), 0.0).clamp(0, 15)
        c = c.nan_to_num(0.0).to(torch.uint8)
        codes[..., 16 * g:16 * g + 16] = c[..., 0::2] + 16 * c[..., 1::2]
        steps[..., 0, g], steps[..., 1, g] = s, m
    return Pages(codes, steps)


def lay(pages, layout):
    """Rows of all heads of a token beside one another, all rows of a head of a page, or parts of wider rows."""
    if layout == "heads":
        return Pages(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in pages))
    if layout == "slice":
        out = []
        for t in pages:
            wide = torch.zeros(t.shape[0], t.shape[1], 2 * t.shape[2], *t.shape[3:], dtype=t.dtype, device=t.device)
            wide[:, :, t.shape[2]:] = t
            out.append(wide[:, :, t.shape[2]:])
        return Pages(*out)
    return Pages(*(t.contiguous() for t in pages))


def make(seed, device, dtype, B, W, H, Hkv, D, ps, positions, lens=None, layout="heads", k_factor=1.0, v_factor=1.0, v_add=0.0, **kw):
    """``paged_cases.make`` with both caches in 4 bits; numbers that nobody may look at have steps of NaN."""
    d = paged_cases.make(seed, "cpu", torch.float32, B, W, H, Hkv, D, ps, positions, lens, **kw)
    for n in ("q", "k", "v"):
        d[n] = d[n].to(dtype)
    d["k_pages"], d["v_pages"] = packed(d.pop("k_cache") * k_factor), packed(d.pop("v_cache") * v_factor + v_add)
    d = {n: Pages(*(t.to(device) for t in x)) if isinstance(x, Pages) else x if x is None else x.to(device) for n, x in d.items()}
    d["q"] = d["q"].transpose(0, 1).contiguous().transpose(0, 1)
    for n in ("k_pages", "v_pages"):
        d[n] = lay(d[n], layout)
    return d


def attention(d, scale=None):
    """→ output, and the average of the magnitudes of the values' two terms, which roundings of the weights are relative to."""
    args = d["table"], d["positions"]
    kw = dict(scale=scale, lens=d["lens"], shared_pages=d["shared_pages"])
    k = values(d["k_pages"])
    return paged_oracle.attention(d["q"], k, values(d["v_pages"]), *args, **kw)[0], paged_oracle.attention(d["q"], k, sizes(d["v_pages"]), *args, **kw)[0]


def bound(dtype, out, size):
    """A half step of the result's own rounding; with 16-bit floats a half step of half precision (2^-11) for each weight and one for each value, which are made
    halves before their product; and what sums, products and exponentials in 32 bits leave: scores are sums of up to 128 products, in parts of magnitude 64 at
    most, off by 128 * 2^-24 * 64 < 2^-11 of them, of which the tests' random signs leave less than a quarter."""
    u = torch.finfo(dtype).eps / 2
    return u * out.abs() + ((2 * 2.0 ** -11 if dtype.itemsize == 2 else 0.0) + 2.0 ** -13) * size + 1e-7


def rotate(x, position, cos, sin, interleaved):
    half = cos.shape[1]
    y = x.double().clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[position, i].double(), sin[position, i].double()
        y[..., a], y[..., b] = x[..., a].double() * c - x[..., b].double() * s, x[..., b].double() * c + x[..., a].double() * s
    return y


def append(q, k, v, positions, cos, sin, slots, tokens, interleaved=False):
    """→ rotated queries, and {slot: (key, value)}, all in 64 bits."""
    B, W = q.shape[:2]
    out, written = torch.zeros(q.shape, dtype=torch.float64), {}
    for b in range(B):
        for w in range(W):
            p, slot = int(positions[b]) + w, int(slots[b, w])
            if 0 <= slot < tokens and 0 <= p < cos.shape[0]:
                out[b, w] = rotate(q[b, w], p, cos, sin, interleaved)
                written[slot] = rotate(k[b, w], p, cos, sin, interleaved), v[b, w].double()
    return out, written


def assign(table, held, free, span, positions, new, ps, lens=None, lengths=None, shared=0, trim=False):
    """→ table, held, free, span, slots as lists, and whether anybody found too few."""
    table, held, free = [list(r) for r in table.tolist()], held.tolist(), free.tolist()
    head, tail = span.tolist()
    n, P, short = len(table[0]) if table else 0, len(free), False
    positions = positions.tolist()
    counts = [0 if p < 0 else new if lens is None else max(0, min(new, int(lens[b]))) for b, p in enumerate(positions)]
    goals = [p + m if m else -1 for p, m in zip(positions, counts)] if lengths is None else lengths.tolist()
    held = [max(shared, min(h, n)) for h in held]
    ring, at, back, asked = list(free), head, tail, 0
    for b, goal in enumerate(goals):
        want = -(-goal // ps) if goal > 0 else 0
        if want > n:
            short = True
        elif want > held[b]:
            asked += want - held[b]
            if asked > tail - head:
                short = True
            else:
                while held[b] < want:
                    table[b][held[b]] = free[at % P]
                    at, held[b] = at + 1, held[b] + 1
        if goal == 0 or (trim and goal > 0):
            keep = max(shared, min(want, n))
            for c in range(keep, held[b]):
                ring[back % P], table[b][c] = table[b][c], -1
                back += 1
            held[b] = min(held[b], keep)
    slots = [[-1] * new for _ in positions]
    for b, p in enumerate(positions):
        for w in range(counts[b]):
            c = (p + w) // ps
            if shared <= c < held[b] and 0 <= table[b][c] < P:
                slots[b][w] = table[b][c] * ps + (p + w) % ps
            else:
                short = True
    return table, held, ring, [at, back], slots, short
