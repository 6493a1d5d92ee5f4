"""Performance cases of serving from a paged key/value cache: new keys and values are rotated and appended to pages, attention reads the
pages (a prefix that the whole batch shares is read once), and drafted tokens are verified against the target's probabilities.

Each case is a plain dict; ``prepare`` builds what a serving program holds before the call (pages, page tables, rotation tables, a
projection's output), ``run`` is one pass, ``work`` counts the bytes and operations that the pass cannot do without, ``exact`` recomputes
it in 64 bits.  Head counts are those of the models in ``models/`` (Llama-2 7B / 13B / 70B, Mixtral, DBRX) and of tensor-parallel shards
of them; tokens and probabilities are random.

Where ``own`` is false, ``run`` computes the operators in elementary torch operations, in 32 bits and rounded once (sums of
probabilities in 64); where it is true, it makes the calls of ``ops.paged`` and ``ops.select`` that a serving program makes.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (query heads, key/value heads): 7B, 13B, 70B, Mixtral, DBRX, one of four shards of 7B, one of eight shards of 70B
HEADS = ((32, 32), (40, 40), (64, 8), (32, 8), (48, 8), (8, 8), (8, 1))
VOCABS = (32000, 32016, 100352)
PAGE_SIZES = (16, 32, 48, 64, 128)
TABLE = 16384           # positions of the rotation tables


def _append(name, batch, new, heads, kv_heads, context, page, dim=128, dtype="bf16", ragged=False):
    c = {"kind": "append", "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "context": context, "page": page,
         "shared": 0, "ragged": ragged, "dtype": dtype}
    return {"name": name, **c} if name else c


def _attention(name, batch, new, heads, kv_heads, context, page, dim=128, dtype="bf16", ragged=False, shared=0):
    c = _append(None, batch, new, heads, kv_heads, context, page, dim, dtype, ragged)
    c.update(kind="shared_attention" if shared else "attention", shared=shared)
    return {"name": name, **c} if name else c


def _verify(name, batch, drafts, vocab, dtype="fp32"):
    c = {"kind": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token of a single conversation: a launch's latency
        _append("append_token", 1, 1, 32, 32, 1000, 16),
        # a drafted window of a busy server, one of eight shards of a 70B model, a half-precision cache
        _append("append_window_fp16", 48, 5, 8, 1, 4000, 32, dtype="fp16"),
        # prompts of unequal length, right-padded, into a fresh cache
        _append("append_prompts", 4, 2000, 64, 8, 2000, 64, ragged=True),
        # one token of a short conversation, batch 1
        _attention("attention_token_short", 1, 1, 32, 8, 300, 16),
        # one token each of a batch of long conversations, of unequal length
        _attention("attention_token_long", 16, 1, 32, 8, 8192, 16),
        # one token each, a key/value head for every query head
        _attention("attention_token_single_heads", 6, 1, 40, 40, 2500, 64),
        # verification of drafted windows of unequal length: five tokens of every sequence
        _attention("attention_window", 8, 5, 64, 8, 6000, 32, ragged=True),
        # a portion of two long prompts behind what the cache holds already; heads of 64 numbers in half precision
        _attention("attention_portion_fp16", 2, 1000, 48, 8, 6000, 128, dim=64, dtype="fp16", ragged=True),
        # a system prompt that every conversation of a large batch begins with, one token each
        _attention("shared_token", 64, 1, 32, 8, 512, 64, shared=4096),
        # the same with drafted windows over a long shared document
        _attention("shared_window", 16, 4, 64, 8, 1000, 16, shared=12288),
        # drafted tokens of one conversation
        _verify("verify_single", 1, 4, 32000),
        # drafted tokens of a busy server, a large vocabulary
        _verify("verify_batch", 64, 7, 100352),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "shared", "verify"])
    if kind == "verify":
        return _verify(None, _log_uniform(rng, 1, 64), rng.randint(1, 7), rng.choice(VOCABS), rng.choice(["fp32", "fp32", "fp32", "bf16"]))
    heads, kv_heads = rng.choice(HEADS)
    page, dim, dtype = rng.choice(PAGE_SIZES), rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"])
    ragged = rng.random() < 0.5
    if kind == "append":
        new = rng.choice([1, rng.randint(2, 8), _log_uniform(rng, 9, 2000)])
        batch = _log_uniform(rng, 1, max(1, min(64, 450000 // (new * (heads + 2 * kv_heads)))))
        return _append(None, batch, new, heads, kv_heads, _log_uniform(rng, new, 2000 + new), page, dim, dtype, ragged)
    if kind == "attention":
        new = rng.choice([1, 1, rng.randint(2, 8), _log_uniform(rng, 9, 1000)])
        batch = _log_uniform(rng, 1, 16 if new <= 8 else 2)
        context = new + _log_uniform(rng, 16, min(6000, 1000000 // (batch * kv_heads)))
        return _attention(None, batch, new, heads, kv_heads, context, page, dim, dtype, ragged)
    new = rng.choice([1, 1, rng.randint(2, 5)])
    batch = _log_uniform(rng, 2, 64 if new == 1 else 16)
    context = new + _log_uniform(rng, 16, min(1000, 200000 // (batch * kv_heads)))
    shared = page * max(1, _log_uniform(rng, 128, 4096) // page)
    return _attention(None, batch, new, heads, kv_heads, context, page, dim, dtype, ragged, shared)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _draws(case, seed):
    """Everything random of a case, from the seed alone."""
    g, c = _generator(seed), case
    if c["kind"] == "verify":
        B, K, V = c["batch"], c["drafts"], c["vocab"]
        logits = torch.randn(B, K + 1, V, generator=g, device=DEVICE) * 2
        noise = torch.randn(B, K, V, generator=g, device=DEVICE) * 0.5
        target = torch.softmax(logits, -1).to(TYPES[c["dtype"]])
        draft = torch.softmax(logits[:, :K] + noise, -1).to(TYPES[c["dtype"]])
        tokens = torch.multinomial(draft.float().view(B * K, V), 1, generator=g).view(B, K)
        return {"tokens": tokens, "draft": draft, "target": target, "accept": torch.rand(B, K, generator=g, device=DEVICE),
                "sample": torch.rand(B, generator=g, device=DEVICE)}
    dtype, B, W, H, G, D, ps = TYPES[c["dtype"]], c["batch"], c["new"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    # tokens in a row's own pages: up to `context`, the new ones among them; a ragged batch has rows of half that and more, and fewer new ones
    own_tokens = torch.randint((max(W, c["context"] // 2)), max(W, c["context"]) + 1, (B,), generator=g, device=DEVICE)
    lens = torch.randint((W + 1) // 2, W + 1, (B,), generator=g, device=DEVICE) if c["ragged"] else None
    positions = c["shared"] + own_tokens - W
    shared, most = c["shared"] // ps, (max(W, c["context"]) + ps - 1) // ps
    pages = shared + B * most + 1                       # the last one belongs to nobody and holds zeros
    order = torch.randperm(pages - 1, generator=g, device=DEVICE).to(torch.int32)
    table = torch.cat([order[:shared].expand(B, shared), order[shared:].view(B, most)], 1).contiguous()
    qkv = _normal(g, dtype, W, B, (H + 2 * G) * D)
    out = {"positions": positions, "lens": lens, "table": table, "shared_pages": order[:shared].clone()}
    if c["kind"] == "append":
        # sections of a fused projection's output, sequences beside one another within a token
        out["q"], out["k"], out["v"] = (s.unflatten(-1, (-1, D)).transpose(0, 1) for s in qkv.split([H * D, G * D, G * D], -1))
        frequencies = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device=DEVICE) / D))
        angles = torch.outer(torch.arange(TABLE, dtype=torch.float64, device=DEVICE), frequencies)
        out["cos"], out["sin"] = angles.cos().float(), angles.sin().float()
    else:
        out["q"] = qkv[..., :H * D].contiguous().unflatten(-1, (H, D)).transpose(0, 1)
    for n in ("k_cache", "v_cache"):
        out[n] = _normal(g, dtype, pages, ps, G, D)
        out[n][-1] = 0
    return out


def prepare(case, seed):
    if own:
        import neuronx_distributed_b200  # noqa: F401
    return {"case": case, **_draws(case, seed)}


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    with torch.no_grad():
        if own:
            from neuronx_distributed_b200 import ops

            s = state
            if kind == "verify":
                return ops.select.verify_drafts(s["tokens"], s["draft"], s["target"], s["accept"], s["sample"])
            if kind == "append":
                q = ops.paged.rope_append(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["table"],
                                          lens=s["lens"])
                return [q, s["k_cache"], s["v_cache"]]
            return ops.paged.attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["positions"], lens=s["lens"],
                                       shared_pages=s["shared_pages"] if kind == "shared_attention" else None)
        return {"verify": _plain_verify, "append": _plain_append, "attention": _plain_attention, "shared_attention": _plain_attention}[kind](state)


def _live(s, W):
    """[B, W]: which of a row's new tokens are none of its padding."""
    w = torch.arange(W, device=DEVICE)
    return (w[None] < s["lens"][:, None]) if s["lens"] is not None else torch.ones(s["positions"].shape[0], W, dtype=torch.bool, device=DEVICE)


def _plain_append(s):
    W, half, ps = s["q"].shape[1], s["q"].shape[3] // 2, s["k_cache"].shape[1]
    live = _live(s, W)
    p = s["positions"][:, None] + torch.arange(W, device=DEVICE)[None]
    cos, sin = s["cos"][p][:, :, None], s["sin"][p][:, :, None]
    alive = live[:, :, None, None]

    def rotate(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return (torch.cat([a * cos - b * sin, b * cos + a * sin], -1) * alive).to(x.dtype)

    # padding goes, as zeros, to the page that belongs to nobody and holds zeros
    page = torch.where(live, torch.gather(s["table"], 1, p // ps).long(), s["k_cache"].shape[0] - 1)
    s["k_cache"][page, p % ps] = rotate(s["k"])
    s["v_cache"][page, p % ps] = s["v"] * alive
    return [rotate(s["q"]), s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    q = s["q"]
    B, W, H, D = q.shape
    ps, G = s["k_cache"].shape[1:3]
    n = s["case"]["shared"] // ps
    live = _live(s, W)
    qg = q.float().view(B, W, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D) * D ** -0.5       # rows: token, head of the group
    own_table = s["table"][:, n:].long()
    k = s["k_cache"][own_table].flatten(1, 2).float().transpose(1, 2)                                     # [B, G, keys, D]
    v = s["v_cache"][own_table].flatten(1, 2).float().transpose(1, 2)
    seen = (torch.arange(k.shape[2], device=DEVICE) + n * ps <= (s["positions"][:, None] + torch.arange(W, device=DEVICE))[..., None])
    scores = (qg @ k.transpose(2, 3)).masked_fill(~seen.repeat_interleave(H // G, 1)[:, None], -math.inf)
    if n:
        # the shared prefix, once for all: every row of the batch against the same keys
        ks = s["k_cache"][s["shared_pages"].long()].flatten(0, 1).float().transpose(0, 1)                 # [G, keys, D]
        vs = s["v_cache"][s["shared_pages"].long()].flatten(0, 1).float().transpose(0, 1)
        rows = qg.transpose(0, 1).reshape(G, -1, D)
        before = (rows @ ks.transpose(1, 2)).view(G, B, -1, n * ps).transpose(0, 1)
        top = torch.maximum(scores.amax(-1, keepdim=True), before.amax(-1, keepdim=True))
        p, pb = torch.exp(scores - top), torch.exp(before - top)
        o = p @ v + (pb.transpose(0, 1).reshape(G, -1, n * ps) @ vs).view(G, B, -1, D).transpose(0, 1)
        o = o / (p.sum(-1, keepdim=True) + pb.sum(-1, keepdim=True))
    else:
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.view(B, G, W, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, W, H, D)
    return (o * live[:, :, None, None]).to(q.dtype)


def _plain_verify(s):
    tokens, B, K = s["tokens"], *s["tokens"].shape
    p = s["target"][:, :K].gather(2, tokens[..., None])[..., 0].double()
    q = s["draft"].gather(2, tokens[..., None])[..., 0].double()
    accepted = (s["accept"].double() * q < p).long().cumprod(1).sum(1)
    rows = torch.arange(B, device=DEVICE)
    weights = s["target"][rows, accepted].double()
    less = s["draft"][rows, accepted.clamp(max=K - 1)].double() * (accepted < K)[:, None]
    rest = (weights - less).clamp(min=0)
    weights = torch.where((rest.sum(1) > 0)[:, None], rest, weights)
    cdf = weights.cumsum(1)
    chosen = (cdf <= s["sample"].double()[:, None] * cdf[:, -1:]).sum(1)
    at = torch.arange(K + 1, device=DEVICE)[None]
    out = torch.where(at < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    return torch.where(at == accepted[:, None], chosen[:, None], out), accepted


# ---------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "verify":
        # a draft is accepted about three times in four; where one is refused, one row of either side is walked, otherwise the target's last
        es = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": es * c["batch"] * c["vocab"] * (2 - 0.75 ** c["drafts"]), "flops": 0}
    es, B, W, H, G, D = TYPES[c["dtype"]].itemsize, c["batch"], c["new"] * (0.75 if c["ragged"] else 1.0), c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        return {"bytes": 2 * es * B * W * (H + 2 * G) * D + 4 * W * D, "flops": 0}
    keys = (c["context"] // 2 + c["context"]) / 2           # sequences stand between half of the context and all of it
    return {"bytes": 2 * es * B * W * H * D + 2 * es * G * D * (B * keys + c["shared"]),
            "flops": 4.0 * B * W * H * D * (max(keys - c["new"] / 2, 1) + c["shared"])}


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    d = _draws(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(d)
    B, W, H, D = d["q"].shape
    ps, G = d["k_cache"].shape[1:3]
    if case["kind"] == "append":
        q_out, kc, vc = torch.zeros(B, W, H, D, dtype=torch.float64, device=DEVICE), d["k_cache"].double(), d["v_cache"].double()
        for b in range(B):
            m = W if d["lens"] is None else int(d["lens"][b])
            at = torch.arange(int(d["positions"][b]), int(d["positions"][b]) + m, device=DEVICE)
            turn = torch.complex(d["cos"][at].double(), d["sin"][at].double())[:, None]
            for x, dst in ((d["q"], q_out[b, :m]), (d["k"], None)):
                z = torch.complex(x[b, :m, :, :D // 2].double(), x[b, :m, :, D // 2:].double()) * turn
                z = torch.cat([z.real, z.imag], -1)
                if dst is None:
                    kc[d["table"][b].long()[at // ps], at % ps] = z
                else:
                    dst.copy_(z)
            vc[d["table"][b].long()[at // ps], at % ps] = d["v"][b, :m].double()
        return [q_out, kc, vc]
    out = torch.zeros(B, W, H, D, dtype=torch.float64, device=DEVICE)
    for b in range(B):
        m = W if d["lens"] is None else int(d["lens"][b])
        end = int(d["positions"][b]) + m
        k = d["k_cache"][d["table"][b].long()].reshape(-1, G, D)[:end].double()
        v = d["v_cache"][d["table"][b].long()].reshape(-1, G, D)[:end].double()
        hidden = torch.arange(end, device=DEVICE)[None] > torch.arange(end - m, end, device=DEVICE)[:, None]
        for h in range(H):
            s = d["q"][b, :m, h].double() @ k[:, h * G // H].T / math.sqrt(D)
            out[b, :m, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h * G // H]
    return out


def _exact_verify(d):
    import numpy as np

    B, K = d["tokens"].shape
    tokens, accept, sample = d["tokens"].tolist(), d["accept"].tolist(), d["sample"].tolist()
    out, counts = [], []
    for b in range(B):
        n = 0
        while n < K and accept[b][n] * float(d["draft"][b, n, tokens[b][n]]) < float(d["target"][b, n, tokens[b][n]]):
            n += 1
        w = d["target"][b, n].double().cpu().numpy()
        if n < K:
            rest = np.maximum(w - d["draft"][b, n].double().cpu().numpy(), 0.0)
            w = rest if rest.sum() > 0 else w
        cdf = np.cumsum(w)
        out.append(tokens[b][:n] + [int(np.searchsorted(cdf, sample[b] * cdf[-1], side="right"))] + [-1] * (K - n))
        counts.append(n)
    return torch.tensor(out, device=DEVICE), torch.tensor(counts, device=DEVICE)
