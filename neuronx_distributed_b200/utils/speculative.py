"""Greedy speculative decoding with a small draft model (reference ``examples/inference/run_llama_speculative.py`` and the
``speculation_length`` path of its model wrapper): the draft proposes ``k`` tokens one by one, the target verifies the
whole window in ONE forward (``speculation_forward``) and accepts the longest matching prefix plus its own next token —
the output is token-for-token identical to the target's greedy decoding.

:func:`speculative_sample` does the same for sampling, over a batch: drafted tokens are drawn from the draft's probabilities and accepted
against the target's (``ops.select.verify_drafts``), so that what comes out is distributed as the target's own samples."""
from __future__ import annotations

from contextlib import ExitStack
from typing import Optional, Tuple

import torch

from .. import ops


def _make_room(ahead: ExitStack, target, draft, rows: int, prompt: int, new: int, window: int) -> int:
    """Pages for ``rows`` sequences in the models whose caches have pages, until ``ahead`` ends → length of the prefix that both models' sequences share."""
    before = [model.kv.shared_tokens if getattr(model, "paged", False) else 0 for model in (target, draft)]
    if before[0] != before[1]:
        raise ValueError(f"the target's shared prefix has {before[0]} tokens, the draft's {before[1]}")
    for model in (target, draft):
        if getattr(model, "paged", False):
            need = before[0] + prompt + new
            ahead.enter_context(model.kv.reserved_ahead(rows, max(need, min(need + window, model.kv.max_seq_len))))
    return before[0]


@torch.no_grad()
def speculative_generate(target, draft, prompt_ids: torch.Tensor, max_new_tokens: int, speculation_length: int = 4
                         ) -> Tuple[torch.Tensor, float]:
    """``target`` / ``draft``: :class:`models.llama_inference.LlamaForInference` with batch size 1 (on-device greedy
    sampling).  Returns ``(generated ids [1, n], mean accepted draft tokens per target forward)``."""
    assert prompt_ids.shape[0] == 1, "speculative decoding example runs batch 1"
    dev = prompt_ids.device
    S = prompt_ids.shape[1]
    with ExitStack() as ahead:
        before = _make_room(ahead, target, draft, 1, S, max_new_tokens, speculation_length)
        t_next = target.context_encoding(prompt_ids)              # token at position S, behind what all sequences share
        draft.context_encoding(prompt_ids)
        out = [int(t_next)]
        pos = before + S                                          # position of the last emitted token (t_next)
        accepted_total, rounds = 0, 0
        while len(out) < max_new_tokens:
            k = min(speculation_length, max_new_tokens - len(out))
            # draft proposes k tokens after t_next
            proposal, tok, p = [], torch.tensor([[out[-1]]], device=dev), pos
            for _ in range(k):
                tok = draft.token_generation(tok.view(1, 1), torch.tensor([p], device=dev)).view(1, 1)
                proposal.append(int(tok))
                p += 1
            # target verifies [t_next, proposal...] in one forward: prediction after each of the k+1 positions
            window = torch.tensor([[out[-1]] + proposal], device=dev)
            pred = target.speculation_forward(window, torch.tensor([pos], device=dev))[0].tolist()     # k+1 tokens
            n_ok = 0
            while n_ok < k and proposal[n_ok] == pred[n_ok]:
                n_ok += 1
            new = proposal[:n_ok] + [pred[n_ok]]
            out.extend(new)
            accepted_total += n_ok
            rounds += 1
            # draft cache: positions pos..pos+k-1 are written ([last token, proposals[:-1]]); rejected entries get overwritten by
            # the next round, but when everything was accepted the last proposal (position pos+k) was never fed to the draft
            if n_ok == k:
                draft.token_generation(torch.tensor([[proposal[-1]]], device=dev), torch.tensor([pos + k], device=dev))
            pos += len(new)
    return torch.tensor([out[:max_new_tokens]], device=dev), accepted_total / max(rounds, 1)


@torch.no_grad()
def speculative_sample(target, draft, prompt_ids: torch.Tensor, max_new_tokens: int, speculation_length: int = 4, temperature: float = 1.0,
                       generator: Optional[torch.Generator] = None, prompt_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, float]:
    """``target`` / ``draft``: :class:`models.llama_inference.LlamaForInference` on one rank, with ``on_device_sampling=False`` (they return logits of
    the whole vocabulary; tensor-parallel ranks have shards of them and are refused), contiguous or paged caches, a shared prefix of the same length in both or none.  ``prompt_ids [B, S]`` (right-padded,
    ``prompt_lens [B]``) → (generated ids ``[B, max_new_tokens]``, mean accepted draft tokens per target forward)."""
    if temperature <= 0:
        raise ValueError(f"temperature must be positive, got {temperature} (greedy decoding: speculative_generate)")
    if speculation_length < 1 or max_new_tokens < 1:
        raise ValueError("speculation_length and max_new_tokens are at least 1")
    if target.on_device_sampling or draft.on_device_sampling:
        raise ValueError("both models have to return logits (on_device_sampling=False)")
    dev, (B, S), K = prompt_ids.device, prompt_ids.shape, speculation_length
    lens = torch.full((B,), S, dtype=torch.long, device=dev) if prompt_lens is None else prompt_lens.long()
    for model in (target, draft):
        most = S + max_new_tokens + K + (model.kv.shared_tokens if getattr(model, "paged", False) else 0)
        if most > model.max_seq_len:
            raise ValueError(f"{most} tokens (shared, prompt, new, window) do not fit max_seq_len {model.max_seq_len}")

    def probabilities(logits):
        if logits.shape[-1] != target.cfg.vocab_size:
            raise ValueError(f"logits of {logits.shape[-1]} tokens, a vocabulary of {target.cfg.vocab_size}: sampled speculation needs whole rows "
                             "(tensor-parallel ranks have shards of them), and one vocabulary")
        return torch.softmax(logits.float() / temperature, -1)

    def uniforms(*shape):
        return torch.rand(*shape, device=dev, generator=generator)

    with ExitStack() as ahead:
        before = _make_room(ahead, target, draft, B, S, max_new_tokens, K)
        tok = torch.multinomial(probabilities(target.context_encoding(prompt_ids, lens - 1)), 1, generator=generator)        # [B, 1]
        draft.context_encoding(prompt_ids, lens - 1)
        pos = lens + before                                       # position of each row's newest token
        rows = [[int(t)] for t in tok[:, 0].tolist()]
        accepted, rounds = 0, 0
        while min(len(r) for r in rows) < max_new_tokens:
            proposal, probs, x = [], [], tok
            for i in range(K):
                probs.append(probabilities(draft.token_generation(x, pos + i)))
                x = torch.multinomial(probs[-1], 1, generator=generator)
                proposal.append(x)
            draft.token_generation(x, pos + K)                    # the last one's keys, should all be accepted
            drafted = torch.cat(proposal, 1)
            judged = probabilities(target.speculation_forward(torch.cat([tok, drafted], 1), pos))
            new, n = ops.select.verify_drafts(drafted, torch.stack(probs, 1), judged, uniforms(B, K), uniforms(B))
            tok = new.gather(1, n[:, None])
            for r, ids, count in zip(rows, new.tolist(), n.tolist()):
                if len(r) < max_new_tokens:
                    r += ids[:count + 1]
                    accepted += count
                    rounds += 1
            # a row that is done goes on in place: nobody reads it
            done = torch.tensor([len(r) >= max_new_tokens for r in rows], device=dev)
            pos = torch.where(done, pos, pos + n + 1)
    return torch.tensor([r[:max_new_tokens] for r in rows], device=dev), accepted / max(rounds, 1)
