"""Row-wise arg-max / top-k on the sm_100a selection kernels (``csrc/select.cu``) with plain PyTorch as the CPU path and the
numerics oracle.  ``index_offset`` shifts the returned indices (global id of a vocab shard's first column)."""
from __future__ import annotations

from typing import Tuple

import torch

from . import _ext


def _kernel_ok(x: torch.Tensor) -> bool:
    return (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16, torch.float32) and x.shape[-1] > 0
            and _ext.ext() is not None and hasattr(_ext.ext(), "row_argmax"))


def row_max(x: torch.Tensor, index_offset: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [..., V] → (max fp32 [...], argmax int64 [...] + index_offset); ties → smallest index."""
    lead = x.shape[:-1]
    if _kernel_ok(x):
        x2 = x.reshape(-1, x.shape[-1])
        if x2.stride(-1) != 1:
            x2 = x2.contiguous()
        _ext.count_launch()
        v, i = _ext.ext().row_argmax(x2, int(index_offset))
        return v.view(lead), i.view(lead)
    v, i = torch.max(x.float(), dim=-1)
    return v, i + index_offset


def row_topk(x: torch.Tensor, k: int, index_offset: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [..., V] → (values fp32 [..., k], indices int64 [..., k] + index_offset), sorted descending."""
    lead = x.shape[:-1]
    V = x.shape[-1]
    if _kernel_ok(x) and _ext.ext().row_topk_supported(V, k):
        x2 = x.reshape(-1, V)
        if x2.stride(-1) != 1:
            x2 = x2.contiguous()
        _ext.count_launch()
        v, i = _ext.ext().row_topk(x2, int(k), int(index_offset))
        return v.view(*lead, k), i.view(*lead, k)
    v, i = torch.topk(x.float(), k, dim=-1)
    return v, i + index_offset


def verify_drafts(draft_tokens: torch.Tensor, draft_probs: torch.Tensor, target_probs: torch.Tensor, accept_uniforms: torch.Tensor,
                  sample_uniforms: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Speculative sampling: drafted tokens against the target's probabilities, from given random numbers in [0, 1) (``csrc/verify.cu``).

    ``draft_tokens [B, K]``, ``draft_probs [B, K, V]`` (what each token was drawn from), ``target_probs [B, K + 1, V]``, ``accept_uniforms [B, K]``,
    ``sample_uniforms [B]`` → (tokens int64 ``[B, K + 1]``, accepted int64 ``[B]``).  Token ``i`` is accepted while ``u_i q_i(x_i) < p_i(x_i)``; behind
    the ``n`` accepted ones comes one drawn from ``max(p_n - q_n, 0)`` (from ``p_K`` when all were accepted): the lowest ``v`` whose running sum of
    weights passes ``sample_uniforms`` of their whole sum; then ``-1``.  A drafted token outside the vocabulary (``-1``: a shorter draft) ends a row's
    draft, and the next one comes from ``p`` itself, as it does where nothing of ``max(p_n - q_n, 0)`` is left.  Rows of probabilities need not sum
    to one; negative ones and NaN count as 0, and a row without any gives ``-1``.  Compared and summed in 64 bits."""
    if torch.is_grad_enabled() and (draft_probs.requires_grad or target_probs.requires_grad):
        raise RuntimeError("verify_drafts has no gradient: call it under torch.no_grad(), or with tensors that ask for none")
    draft_tokens, accept_uniforms, sample_uniforms = draft_tokens.contiguous(), accept_uniforms.contiguous(), sample_uniforms.contiguous()
    if _ext.use_cuda(target_probs):
        return tuple(_ext.ext().verify_drafts(draft_tokens, draft_probs, target_probs, accept_uniforms, sample_uniforms))

    def need(ok, text):
        if not ok:
            raise ValueError(text)

    need(draft_tokens.dim() == 2 and draft_tokens.dtype == torch.long, "draft_tokens must be a contiguous int64 tensor [batch, drafts]")
    B, K = draft_tokens.shape
    need(draft_probs.dim() == 3 and target_probs.dim() == 3 and draft_probs.shape[:2] == (B, K) and target_probs.shape[:2] == (B, K + 1)
         and draft_probs.shape[2] == target_probs.shape[2] and target_probs.shape[2] > 0,
         "probabilities must be [batch, drafts, vocabulary] of the draft and [batch, drafts + 1, vocabulary] of the target, got "
         f"{tuple(draft_probs.shape)} and {tuple(target_probs.shape)}")
    need(draft_probs.dtype == target_probs.dtype and target_probs.dtype in (torch.float32, torch.bfloat16, torch.float16),
         "probabilities are float32, bfloat16 or float16, both of one type")
    need(accept_uniforms.shape == draft_tokens.shape and accept_uniforms.dtype == torch.float32,
         "accept_uniforms must be a contiguous float32 tensor [batch, drafts]")
    need(sample_uniforms.shape == (B,) and sample_uniforms.dtype == torch.float32, "sample_uniforms must be a contiguous float32 tensor [batch]")
    need(all(t.device == target_probs.device for t in (draft_tokens, draft_probs, accept_uniforms, sample_uniforms)), "all tensors are on one device")
    V = target_probs.shape[2]
    rows = torch.arange(B, device=target_probs.device)
    there = (draft_tokens >= 0) & (draft_tokens < V)
    at = draft_tokens.clamp(0, V - 1)[..., None]
    zero = lambda x: torch.where(x > 0, x, 0.0)               # negative numbers and NaN count as 0

    ok = there & (accept_uniforms.double() * zero(draft_probs.gather(2, at)[..., 0].double()) < target_probs[:, :K].gather(2, at)[..., 0].double())
    n = ok.long().cumprod(1).sum(1)
    p = target_probs[rows, n].double()
    w = p
    if K:
        residual = (n < K) & there.gather(1, n.clamp(max=K - 1)[:, None])[:, 0]
        w = p - torch.where(residual[:, None], zero(draft_probs[rows, n.clamp(max=K - 1)].double()), 0.0)
    w = zero(w)
    w = torch.where((w.sum(1) > 0)[:, None], w, zero(p))
    cdf = w.cumsum(1)
    hit = (w > 0) & (cdf > sample_uniforms.double()[:, None] * cdf[:, -1:])
    index = torch.arange(V, device=w.device)
    first = torch.where(hit, index, V).amin(1)
    chosen = torch.where(first < V, first, torch.where(w > 0, index, -1).amax(1))
    slot = torch.arange(K + 1, device=w.device)[None]
    kept = torch.cat([draft_tokens, draft_tokens.new_full((B, 1), -1)], 1)
    return torch.where(slot < n[:, None], kept, torch.where(slot == n[:, None], chosen[:, None], -1)), n
