"""Random inputs of the paged operators: pages in no order, garbage wherever nobody may look."""
import torch


def make(seed, device, dtype, B, W, H, Hkv, D, ps, positions, lens=None, shared=0, cols=None, spare=3, garbage=float("nan"), layout="rows"):
    """``positions`` (of the first new token, negative: idle), ``lens`` as lists; ``shared`` pages in common.  Pages that belong to nobody and rows
    behind a sequence's last token hold ``garbage``.  ``layout``: pages of ``rows`` or ``heads`` first, or a ``slice`` of wider rows."""
    g = torch.Generator().manual_seed(seed)
    pos = torch.tensor(positions, dtype=torch.long)
    n_new = torch.full((B,), W) if lens is None else torch.tensor(lens).clamp(0, W)
    ends = torch.where(pos < 0, 0, pos + n_new)
    most = max(int(ends.max()), 1)
    cols = (most + ps - 1) // ps if cols is None else cols
    cols = max(cols, shared)
    pages = shared + B * (cols - shared) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.empty(B, cols, dtype=torch.int32)
    table[:, :shared] = order[:shared].to(torch.int32)
    table[:, shared:] = order[shared:shared + B * (cols - shared)].view(B, -1).to(torch.int32)
    rnd = lambda *s: torch.randn(*s, generator=g)
    kc, vc = rnd(pages, ps, Hkv, D), rnd(pages, ps, Hkv, D)
    used = torch.zeros(pages, ps, dtype=torch.bool)
    for b in range(B):
        for j in range(min(int(ends[b]), cols * ps)):
            used[table[b, j // ps].long(), j % ps] = True
    if shared:
        used[table[0, :shared].long()] = True
    kc[~used] = garbage
    vc[~used] = garbage
    q = rnd(W, B, H, D).transpose(0, 1)
    k, v = rnd(B, W, Hkv, D), rnd(B, W, Hkv, D)
    move = lambda t: t.to(dtype).to(device)

    def cache(t):
        t = move(t)
        if layout == "heads":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "slice":
            wide = torch.zeros(pages, ps, Hkv, 2 * D, dtype=dtype, device=device)
            wide[..., D:] = t
            return wide[..., D:]
        return t

    return {"q": move(q), "k": move(k), "v": move(v), "k_cache": cache(kc), "v_cache": cache(vc), "table": table.to(device),
            "positions": pos.to(device), "lens": None if lens is None else torch.tensor(lens, dtype=torch.long, device=device),
            "shared_pages": table[0, :shared].clone().to(device) if shared else None}


def bound(dtype, out, size):
    """A half step of the result's own rounding, a half step of every weight's (both ``eps / 2`` relative), and what sums, products and
    exponentials in 32 bits leave: scores are sums of up to 128 products of about 10 in all, off by 128 * 2^-24 * 10 < 2^-13 of the weights at worst."""
    u = torch.finfo(dtype).eps / 2
    return u * out.abs() + (u + 2.0 ** -13) * size + 1e-7
