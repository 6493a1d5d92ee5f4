"""The operators of a paged cache from their definitions, in 64 bits, one sequence and one token at a time."""
import math

import torch


def rotate(x, position, cos, sin):
    """``x [..., D]`` at one position."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half].double(), x[..., half:].double(), cos[position].double(), sin[position].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def new_tokens(W, positions, lens, b):
    if int(positions[b]) < 0:
        return 0
    return W if lens is None else max(0, min(W, int(lens[b])))


def append(q, k, v, positions, cos, sin, k_cache, v_cache, table, lens=None):
    """→ rotated queries, keys and values as they stand afterwards, and where something was written ``[pages, page_size]``."""
    B, W, H, D = q.shape
    pages, ps = k_cache.shape[:2]
    out = torch.zeros(B, W, H, D, dtype=torch.float64, device=q.device)
    kc, vc = k_cache.double(), v_cache.double()
    written = torch.zeros(pages, ps, dtype=torch.bool)
    for b in range(B):
        for w in range(new_tokens(W, positions, lens, b)):
            p = int(positions[b]) + w
            if p >= cos.shape[0]:
                continue
            out[b, w] = rotate(q[b, w], p, cos, sin)
            page = int(table[b, p // ps]) if p // ps < table.shape[1] else -1
            if 0 <= page < pages:
                kc[page, p % ps] = rotate(k[b, w], p, cos, sin)
                vc[page, p % ps] = v[b, w].double()
                written[page, p % ps] = True
    return out, kc, vc, written


def attention(q, k_cache, v_cache, table, positions, scale=None, lens=None, shared_pages=None):
    """→ output, and the same average of the values' magnitudes, which roundings of the weights are relative to."""
    B, W, H, D = q.shape
    pages, ps, Hkv, _ = k_cache.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, W, H, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for b in range(B):
        row = table[b].tolist()
        if shared_pages is not None:
            row = shared_pages.tolist() + row[len(shared_pages):]
        m = new_tokens(W, positions, lens, b)
        end = min(int(positions[b]) + m, len(row) * ps)
        at = [(row[j // ps], j % ps) if 0 <= row[j // ps] < pages else None for j in range(end)] if m else []
        there = torch.tensor([a is not None for a in at], dtype=torch.bool, device=q.device)
        page = torch.tensor([a[0] if a else 0 for a in at], dtype=torch.long, device=q.device)
        slot = torch.tensor([a[1] if a else 0 for a in at], dtype=torch.long, device=q.device)
        keys = torch.where(there[:, None, None], k_cache[page, slot].double(), 0.0)
        values = torch.where(there[:, None, None], v_cache[page, slot].double(), 0.0)
        for w in range(m):
            n = min(int(positions[b]) + w + 1, end)
            seen = there[:n]
            if not bool(seen.any()):
                continue
            for h in range(H):
                g = h // (H // Hkv)
                s = (keys[:n, g] @ q[b, w, h].double() * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(s, 0)
                out[b, w, h] = p @ values[:n, g]
                size[b, w, h] = p @ values[:n, g].abs()
    return out, size


def verify(tokens, draft, target, accept, sample):
    B, K = tokens.shape
    V = target.shape[2]
    out, counts = [], []
    for b in range(B):
        n, there = 0, True
        while n < K:
            x = int(tokens[b, n])
            there = 0 <= x < V
            if not there or not float(accept[b, n]) * float(draft[b, n, x]) < float(target[b, n, x]):
                break
            n += 1
        p = [float(x) for x in target[b, n]]
        w = list(p)
        if n < K and there:
            w = [x - float(y) for x, y in zip(p, draft[b, n])]
        w = [x if x > 0 else 0.0 for x in w]
        if not sum(w) > 0:
            w = [x if x > 0 else 0.0 for x in p]
        total, run, chosen = math.fsum(w), 0.0, -1
        for i, x in enumerate(w):
            if x > 0:
                chosen = i
                run = math.fsum(w[:i + 1]) if V < 64 else run + x
                if run > float(sample[b]) * total:
                    break
        out.append([int(t) for t in tokens[b, :n]] + [chosen] + [-1] * (K - n))
        counts.append(n)
    return torch.tensor(out), torch.tensor(counts)
