"""Performance cases of serving from a paged key/value cache that is held in 4 bits: page tables and slots of new tokens from the requests' lengths,
new keys and values rotated, rounded to codes and written to their slots, and attention over the codes.

Each case is a plain dict; ``prepare`` builds what a serving program holds before the call (pages, tables, rotation tables, a projection's output),
``run`` is one pass, ``work`` counts the bytes and operations that the pass cannot do without, ``exact`` recomputes it in 64 bits.  Head counts are
those of the models in ``models/`` (Llama-2 7B / 13B / 70B, Mixtral, DBRX) and of tensor-parallel shards of them; tokens are random.

A group of 32 numbers of a token's head is held as ``m + s c``: ``m`` and ``s`` in half precision, the least of them and a fifteenth of their range, and codes
``c`` of 0 to 15.  An append returns the rotated queries and what the cache then holds for the new tokens, in the model's type.

Where ``own`` is false, ``run`` computes the operators in elementary torch operations, in 32 bits and rounded once (codes, which stand next to borders,
from 64); where it is true, it makes the calls of ``ops.page_tables`` and ``ops.paged_int4`` that a serving program makes.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32
# (query heads, key/value heads): 7B, 13B, 70B, Mixtral, DBRX, one of four shards of 7B, one of eight shards of 70B
HEADS = ((32, 32), (40, 40), (64, 8), (32, 8), (48, 8), (8, 8), (8, 1))
PAGE_SIZES = (16, 32, 48, 64, 128)
ROTATIONS = ("halves", "halves", "pairs", "part", "part_pairs")         # the whole head or half of it, halves or neighbours
TABLE = 16384           # positions of the rotation tables


def _append(name, batch, new, heads, kv_heads, page, dim=128, dtype="bf16", ragged=False, rotation="halves"):
    c = {"kind": "append", "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged,
         "rotation": rotation, "dtype": dtype}
    return {"name": name, **c} if name else c


def _attention(name, batch, new, heads, kv_heads, context, page, dim=128, dtype="bf16", ragged=False):
    c = {"kind": "attention", "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "context": context, "page": page,
         "ragged": ragged, "dtype": dtype}
    return {"name": name, **c} if name else c


def _tables(name, batch, new, context, page, turnover=False, shared=0):
    c = {"kind": "tables", "batch": batch, "new": new, "context": context, "page": page, "turnover": turnover, "shared": shared}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token of a single conversation: a launch's latency
        _append("append_token", 1, 1, 32, 32, 16),
        # a drafted window of a busy server, half of each head rotated in neighbouring pairs, half precision
        _append("append_window_fp16", 48, 5, 48, 8, 32, dim=64, dtype="fp16", rotation="part_pairs"),
        # prompts of unequal length, right-padded
        _append("append_prompts", 4, 2000, 64, 8, 64, ragged=True),
        # one token of a short conversation, batch 1
        _attention("attention_token_short", 1, 1, 32, 8, 300, 16),
        # one token each of a batch of long conversations, of unequal length
        _attention("attention_token_long", 16, 1, 32, 8, 8192, 16),
        # one token each, a key/value head for every query head
        _attention("attention_token_single_heads", 6, 1, 40, 40, 2500, 64),
        # one token behind a whole book
        _attention("attention_token_book", 1, 1, 64, 8, 100000, 128),
        # verification of drafted windows of unequal length in half precision: five tokens of every sequence
        _attention("attention_window_fp16", 8, 5, 64, 8, 6000, 32, dtype="fp16", ragged=True),
        # a portion of two long prompts behind what the cache holds already, heads of 64 numbers
        _attention("attention_portion", 2, 1000, 48, 8, 6000, 128, dim=64, ragged=True),
        # one new token each of a batch of conversations, some of which begin a page
        _tables("tables_token", 16, 1, 4000, 16),
        # a turn of a batch: conversations end, others begin with prompts behind a shared prefix, the rest goes on
        _tables("tables_turnover", 64, 2000, 6000, 16, turnover=True, shared=1024),
        # one new token each of a very large batch of long conversations
        _tables("tables_token_large", 2000, 1, 32000, 16),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "tables"])
    page = rng.choice(PAGE_SIZES)
    if kind == "tables":
        turnover = rng.random() < 0.5
        new = _log_uniform(rng, 9, 2000) if turnover else rng.choice([1, rng.randint(2, 8)])
        batch = _log_uniform(rng, 1, min(2000, 128000 // new))
        context = new + _log_uniform(rng, 16, min(32000, 60000000 // batch))
        return _tables(None, batch, new, context, page, turnover, page * rng.randint(0, min(64, (context - new) // page)))
    heads, kv_heads = rng.choice(HEADS)
    dim, dtype, ragged = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.5
    if kind == "append":
        new = rng.choice([1, rng.randint(2, 8), _log_uniform(rng, 9, 2000)])
        batch = _log_uniform(rng, 1, max(1, min(64, 500000 // (new * (heads + 2 * kv_heads)))))
        return _append(None, batch, new, heads, kv_heads, page, dim, dtype, ragged, rng.choice(ROTATIONS))
    new = rng.choice([1, 1, rng.randint(2, 8), _log_uniform(rng, 9, 1000)])
    batch = _log_uniform(rng, 1, 16 if new <= 8 else 2)
    context = new + _log_uniform(rng, 16, max(17, min(100000, 1000000 // (batch * kv_heads), 30000000000 // (batch * new * heads * dim) - new)))
    return _attention(None, batch, new, heads, kv_heads, context, page, dim, dtype, ragged)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEVICE)


def _pages(g, pages, page, heads, dim):
    """Codes and steps of random numbers: ``[pages, page, heads, dim / 2]`` bytes and ``[pages, page, heads, 2, dim / 32]`` in half precision, the rows of
    a page's head beside one another in memory; the last page holds zeros."""
    x = torch.randn(pages, heads, page, dim // GROUP, GROUP, generator=g, device=DEVICE)
    lo = x.amin(-1).half()
    s = ((x.amax(-1) - lo.float()) / 15).half()
    c = ((x - lo.float()[..., None]) / s.float()[..., None]).round_().clamp_(0, 15).to(torch.uint8).flatten(-2)
    del x
    codes, steps = c[..., ::2] | c[..., 1::2] << 4, torch.stack([s, lo], -2)
    codes[-1], steps[-1] = 0, 0
    return codes.transpose(1, 2), steps.transpose(1, 2)


def _draws(case, seed):
    """Everything random of a case, from the seed alone."""
    g, c = _generator(seed), case
    if c["kind"] == "tables":
        return _draw_tables(g, c)
    dtype, B, W, H, G, D, ps = TYPES[c["dtype"]], c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    lens = _ints(g, (W + 1) // 2, W, B) if c["ragged"] else None
    if c["kind"] == "append":
        # sections of a fused projection's output, sequences beside one another within a token
        out = {"lens": lens, "positions": _ints(g, 0, TABLE - W, B)}
        qkv = _normal(g, dtype, W, B, (H + 2 * G) * D)
        out["q"], out["k"], out["v"] = (s.unflatten(-1, (-1, D)).transpose(0, 1) for s in qkv.split([H * D, G * D, G * D], -1))
        rotated = D // 2 if c["rotation"].startswith("part") else D
        angles = torch.outer(torch.arange(TABLE, dtype=torch.float64, device=DEVICE),
                             1.0 / (10000.0 ** (torch.arange(0, rotated, 2, dtype=torch.float64, device=DEVICE) / rotated)))
        out["cos"], out["sin"] = angles.cos().float(), angles.sin().float()
        # a page more than the tokens fill, for each sequence; the last one belongs to nobody
        most = (W + ps - 1) // ps + 1
        pages = B * most + 1
        table = torch.randperm(pages - 1, generator=g, device=DEVICE).view(B, most)
        at = _ints(g, 0, ps - 1, B)[:, None] + torch.arange(W, device=DEVICE)
        slots = table.gather(1, at // ps) * ps + at % ps
        if lens is not None:
            slots = torch.where(torch.arange(W, device=DEVICE) < lens[:, None], slots, -1)
        out["slots"] = slots.int()
    else:
        keys = _ints(g, max(W, c["context"] // 2), max(W, c["context"]), B)
        most = (max(W, c["context"]) + ps - 1) // ps
        pages = B * most + 1
        out = {"lens": lens, "positions": keys - W,
               "table": torch.randperm(pages - 1, generator=g, device=DEVICE).int().view(B, most),
               "q": _normal(g, dtype, W, B, H * D).unflatten(-1, (H, D)).transpose(0, 1)}
    out["k_codes"], out["k_steps"] = _pages(g, pages, ps, G, D)
    out["v_codes"], out["v_steps"] = _pages(g, pages, ps, G, D)
    return out


def _draw_tables(g, c):
    B, W, ps, shared = c["batch"], c["new"], c["page"], c["shared"] // c["page"]
    n = (c["context"] + ps - 1) // ps
    pages = B * (n - shared) + shared
    tokens = _ints(g, max(c["shared"], c["context"] // 2), c["context"], B)      # of all rows after this step
    held = ((tokens - (0 if c["turnover"] else W)).clamp(min=c["shared"]) + ps - 1) // ps
    lengths, positions, lens = None, tokens - W, None
    if c["turnover"]:
        # a third of the rows ends, a third begins, the others have no new tokens in this step
        what = _ints(g, 0, 2, B)
        lens = _ints(g, (W + 1) // 2, W, B)
        held = torch.where(what == 1, shared, held)
        lengths = torch.where(what == 0, 0, torch.where(what == 1, c["shared"] + lens, -1))
        positions = torch.where(what == 1, c["shared"], -1)
        fresh = (lengths + ps - 1) // ps > n
        lengths, positions = torch.where(fresh, -1, lengths), torch.where(fresh, -1, positions)
    else:
        positions = torch.where(positions < c["shared"], -1, positions)
        positions[_ints(g, 0, B - 1, B // 16)] = -1                               # idle rows
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    column = torch.arange(n, device=DEVICE)
    own = order[shared:].view(B, n - shared)
    table = torch.cat([order[:shared].expand(B, shared), own], 1)
    table = torch.where(column < held[:, None], table, -1).contiguous()
    # the free pages in a random order, as far round the ring as past steps have brought it
    mine = (column[shared:] >= held[:, None]).flatten()
    first = _ints(g, 0, pages - 1, 1)
    ring = torch.full((pages + 1,), -1, dtype=torch.int32, device=DEVICE)
    ring[torch.where(mine, (first + mine.cumsum(0) - 1) % pages, pages)] = own.flatten()
    span = torch.cat([first, first + mine.sum()])
    return {"table": table, "held": held.int(), "free": ring[:pages].clone(), "span": span, "lengths": lengths, "positions": positions, "lens": lens}


def prepare(case, seed):
    if own:
        import neuronx_distributed_b200  # noqa: F401
    return {"case": case, **_draws(case, seed)}


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    with torch.no_grad():
        if own:
            from neuronx_distributed_b200 import ops

            if c["kind"] == "tables":
                return ops.page_tables.assign(s["table"], s["held"], s["free"], s["span"], s["positions"], c["new"], c["page"], lens=s["lens"],
                                              lengths=s["lengths"], shared=c["shared"] // c["page"])
            k, v = ops.paged_int4.Pages(s["k_codes"], s["k_steps"]), ops.paged_int4.Pages(s["v_codes"], s["v_steps"])
            if c["kind"] == "append":
                q = ops.paged_int4.append(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], k, v, s["slots"],
                                          interleaved=c["rotation"].endswith("pairs"))
                return [q, *ops.paged_int4.gather(k, v, s["slots"], s["q"].dtype)]
            return ops.paged_int4.attention(s["q"], k, v, s["table"], s["positions"], lens=s["lens"])
        return {"append": _plain_append, "attention": _plain_attention, "tables": _plain_tables}[c["kind"]](s)


def _plain_append(s):
    B, W, H, D = s["q"].shape
    slots, half, pairs, ps = s["slots"].long(), s["cos"].shape[1], s["case"]["rotation"].endswith("pairs"), s["k_codes"].shape[1]
    live = slots >= 0
    p = (s["positions"][:, None] + torch.arange(W, device=DEVICE)).clamp(max=TABLE - 1)
    cos, sin = s["cos"][p][:, :, None].double(), s["sin"][p][:, :, None].double()

    def rotate(x):
        t, rest = x[..., :2 * half].double(), x[..., 2 * half:].double()
        a, b = (t[..., ::2], t[..., 1::2]) if pairs else (t[..., :half], t[..., half:])
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1 if pairs else -2).flatten(-2)
        return torch.cat([y, rest], -1)

    # tokens without a slot go, as zeros, to the page that belongs to nobody and holds zeros
    at = torch.where(live, slots, s["k_codes"].shape[0] * ps - 1)
    page, row = at // ps, at % ps
    out = [(rotate(s["q"]) * live[:, :, None, None]).to(s["q"].dtype)]
    for x, codes, steps in ((rotate(s["k"]), s["k_codes"], s["k_steps"]), (s["v"].double(), s["v_codes"], s["v_steps"])):
        x = (x * live[:, :, None, None]).unflatten(-1, (-1, GROUP))
        lo = x.amin(-1).half()
        step = ((x.amax(-1) - lo.double()) / 15).half()
        c = ((x - lo.double()[..., None]) / step.double()[..., None]).round().clamp(0, 15)
        c = torch.where(step[..., None] > 0, c, 0.0).to(torch.uint8).flatten(-2)
        codes[page, row] = c[..., ::2] | c[..., 1::2] << 4
        steps[page, row] = torch.stack([step, lo], -2)
        out.append((_values(codes[page, row], steps[page, row]) * live[:, :, None, None]).to(s["q"].dtype))
    return out


def _values(codes, steps):
    """What codes and steps stand for, in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (c * steps[..., 0, :, None].float() + steps[..., 1, :, None].float()).flatten(-2)


def _plain_attention(s):
    q, table = s["q"], s["table"].long()
    B, W, H, D = q.shape
    G = s["k_codes"].shape[2]
    qg = q.float().view(B, W, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D) * D ** -0.5       # rows: token, head of the group
    k = _values(s["k_codes"][table], s["k_steps"][table]).flatten(1, 2).transpose(1, 2)                   # [B, G, keys, D]
    v = _values(s["v_codes"][table], s["v_steps"][table]).flatten(1, 2).transpose(1, 2)
    w = torch.arange(W, device=DEVICE)
    seen = torch.arange(k.shape[2], device=DEVICE) <= (s["positions"][:, None] + w)[..., None]
    scores = (qg @ k.transpose(2, 3)).masked_fill(~seen.repeat_interleave(H // G, 1)[:, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.view(B, G, W, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, W, H, D)
    return (o if s["lens"] is None else o * (w < s["lens"][:, None])[..., None, None]).to(q.dtype)


def _plain_tables(s):
    c, table, held, free = s["case"], s["table"], s["held"].long(), s["free"]
    (B, n), P, W, ps, shared = table.shape, free.shape[0], c["new"], c["page"], c["shared"] // c["page"]
    counts = torch.where(s["positions"] < 0, 0, W if s["lens"] is None else s["lens"])
    lengths = torch.where(counts > 0, s["positions"] + counts, -1) if s["lengths"] is None else s["lengths"]
    want = (lengths + ps - 1) // ps
    take = torch.where((lengths > 0) & (want <= n), (want - held).clamp(min=0), 0)
    upto = take.cumsum(0)
    take = torch.where(upto <= s["span"][1] - s["span"][0], take, 0)
    give = torch.where(lengths == 0, (held - shared).clamp(min=0), 0)
    back = give.cumsum(0) - give
    column = torch.arange(n, device=DEVICE)
    taken = (column >= held[:, None]) & (column < (held + take)[:, None])
    given = (column >= (held - give)[:, None]) & (column < held[:, None])
    fresh = free[(s["span"][0] + (upto - take)[:, None] + column - held[:, None]) % P]
    new_table = torch.where(taken, fresh, torch.where(given, -1, table))
    place = torch.where(given, (s["span"][1] + back[:, None] + column - (held - give)[:, None]) % P, P)
    new_free = torch.cat([free, free[:1]]).scatter_(0, place.flatten(), table.flatten())[:P]
    p = s["positions"][:, None] + torch.arange(W, device=DEVICE)
    at = (p // ps).clamp(0, n - 1)
    page = new_table.gather(1, at)
    has = (torch.arange(W, device=DEVICE) < counts[:, None]) & (p < n * ps) & (at >= shared) & (page >= 0) & (page < P)
    slots = torch.where(has, page * ps + p % ps, -1).int()
    return [new_table, (held + take - give).int(), new_free, s["span"] + torch.stack([take.sum(), give.sum()]), slots]


# ---------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "tables":
        # the table and the ring, read and written, the rows' numbers, and the slots; rows that go on have no new tokens in a turnover
        B, n, shared = c["batch"], -(-c["context"] // c["page"]), c["shared"] // c["page"]
        return {"bytes": 8.0 * B * n + 8.0 * (B * (n - shared) + shared) + 24.0 * B + 4.0 * B * c["new"], "flops": 0}
    B, W, H, G, D = c["batch"], c["new"] * (0.75 if c["ragged"] else 1.0), c["heads"], c["kv_heads"], c["dim"]
    row = D / 2 + D / 8                                     # bytes of a key or a value in the cache
    if c["kind"] == "append":
        # queries in and out, keys and values in, to the cache, and read from there again
        return {"bytes": 4.0 * B * W * H * D + 2 * B * W * G * (4.0 * D + 2 * row) + 4 * W * D, "flops": 0}
    keys = (c["context"] // 2 + c["context"]) / 2           # sequences stand between half of the context and all of it
    return {"bytes": 4.0 * B * W * H * D + 2 * row * G * B * keys, "flops": 4.0 * B * W * H * D * max(keys - c["new"] / 2, 1)}


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    d = _draws(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "tables": _exact_tables}[case["kind"]](d, case)


def _exact_append(d, c):
    B, W, H, D = d["q"].shape
    G, half = d["k"].shape[2], d["cos"].shape[1]
    out = [torch.zeros(B, W, heads, D, dtype=torch.float64, device=DEVICE) for heads in (H, G, G)]
    for b in range(B):
        m = W if d["lens"] is None else int(d["lens"][b])
        at = int(d["positions"][b])
        turn = torch.complex(d["cos"][at:at + m].double(), d["sin"][at:at + m].double())[:, None]
        turned = []
        for x in (d["q"][b, :m].double(), d["k"][b, :m].double()):
            x = x.clone()
            first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["rotation"].endswith("pairs") else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            turned.append(x)
        out[0][b, :m] = turned[0]
        for dst, x in ((out[1], turned[1]), (out[2], d["v"][b, :m].double())):
            for g in range(0, D, GROUP):
                part = x[..., g:g + GROUP]
                lo = part.min(-1, keepdim=True).values.half().double()
                step = ((part.max(-1, keepdim=True).values - lo) / 15).half().double()
                dst[b, :m, :, g:g + GROUP] = lo + step * torch.round((part - lo) / step).clamp(0, 15)
    return out


def _exact_attention(d, c):
    B, W, H, D = d["q"].shape
    G = d["k_codes"].shape[2]
    out = torch.zeros(B, W, H, D, dtype=torch.float64, device=DEVICE)
    for b in range(B):
        m = W if d["lens"] is None else int(d["lens"][b])
        end = int(d["positions"][b]) + W                    # the row's keys; the last of them belong to padding where there is any
        hidden = torch.arange(end, device=DEVICE)[None] > torch.arange(end - W, end - W + m, device=DEVICE)[:, None]
        for g in range(G):
            side = []
            for codes, steps in ((d["k_codes"], d["k_steps"]), (d["v_codes"], d["v_steps"])):
                code = codes[d["table"][b].long(), :, g].reshape(-1, D // 2)[:end]
                step = steps[d["table"][b].long(), :, g].reshape(-1, 2, D // GROUP)[:end].double().repeat_interleave(GROUP, -1)
                x = torch.empty(end, D, dtype=torch.float64, device=DEVICE)
                x[:, ::2], x[:, 1::2] = (code % 16).double(), (code // 16).double()
                side.append(step[:, 1] + step[:, 0] * x)
            for h in range(g * H // G, (g + 1) * H // G):
                s = d["q"][b, :m, h].double() @ side[0].T / math.sqrt(D)
                out[b, :m, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ side[1]
    return out


def _exact_tables(d, c):
    table, held, free = (d[n].cpu().tolist() for n in ("table", "held", "free"))
    head, tail = d["span"].tolist()
    W, ps, shared, P, n = c["new"], c["page"], c["shared"] // c["page"], len(free), len(table[0])
    positions = d["positions"].tolist()
    counts = [0 if p < 0 else W if d["lens"] is None else int(d["lens"][b]) for b, p in enumerate(positions)]
    lengths = [p + m if m else -1 for p, m in zip(positions, counts)] if d["lengths"] is None else d["lengths"].tolist()
    new_free, at, back, needed = list(free), head, tail, 0
    for b, length in enumerate(lengths):
        want = -(-length // ps)
        if length == 0:
            while held[b] > shared:                         # in the order of the columns
                pages, table[b][shared:held[b]] = table[b][shared:held[b]], [-1] * (held[b] - shared)
                for page in pages:
                    new_free[back % P] = page
                    back += 1
                held[b] = shared
        elif held[b] < want <= n:
            needed += want - held[b]
            if needed <= tail - head:
                for column in range(held[b], want):
                    table[b][column] = free[at % P]
                    at += 1
                held[b] = want
    slots = []
    for b, p in enumerate(positions):
        row = [-1] * W
        for w in range(counts[b]):
            column = (p + w) // ps
            if shared <= column < n and table[b][column] >= 0:
                row[w] = table[b][column] * ps + (p + w) % ps
        slots.append(row)
    whole = lambda v, t: torch.tensor(v, dtype=t, device=DEVICE)  # noqa: E731
    return [whole(table, torch.int32), whole(held, torch.int32), whole(new_free, torch.int32), whole([at, back], torch.int64), whole(slots, torch.int32)]
