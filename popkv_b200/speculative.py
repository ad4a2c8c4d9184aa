"""Verification of drafted tokens (speculative decoding).

``verify_drafts`` decides, on the device and without a host round trip, how many of each
sequence's drafted tokens the target model keeps and which token follows them.  The accepted
tokens and the following one are distributed exactly as the target's own samples.

The reference decodes one token per call (popkv.py:988-1115) and has no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                  noise: torch.Tensor, *, draft_probs: torch.Tensor | None = None,
                  counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Accept drafted tokens against the target's probabilities, from given random numbers.

    Args:
        target_probs: fp32/fp16/bf16 [n, drafts + 1, vocab], the target's probabilities at each
            drafted token's place and after the last.
        draft_tokens: int64 [n, drafts].
        uniforms: fp32 [n, drafts], U[0, 1).
        noise: fp32 [n, vocab], Exp(1) (positive).
        draft_probs: the proposal's probabilities [n, drafts, vocab] in target_probs' type; None for
            drafts that were not drawn at random (greedy or looked up).
        counts: int32 [n], drafts of each sequence (default all); row j = counts[i] of target_probs
            follows the last one.

    Draft j is accepted while ``uniforms * q(draft) < p(draft)``.  The following token wins the race
    ``argmax weight / noise`` over weight > 0, weight = max(p - q, 0) at the first refusal (p where
    that is zero everywhere) and p after the last draft; ties go to the lowest id.

    Returns (tokens int64 [n, drafts + 1]: accepted drafts, the following token, then -1; accepted
    int32 [n]).
    """
    if target_probs.ndim != 3 or draft_tokens.ndim != 2:
        raise ValueError("target_probs must be [n, drafts + 1, vocab] and draft_tokens [n, drafts]")
    n, drafts = (int(x) for x in draft_tokens.shape)
    vocab = int(target_probs.shape[2])
    if tuple(target_probs.shape[:2]) != (n, drafts + 1) or vocab < 1:
        raise ValueError("target_probs must be [n, drafts + 1, vocab]")
    if tuple(uniforms.shape) != (n, drafts) or tuple(noise.shape) != (n, vocab):
        raise ValueError("uniforms must be [n, drafts] and noise [n, vocab]")
    if draft_probs is not None and tuple(draft_probs.shape) != (n, drafts, vocab):
        raise ValueError("draft_probs must be [n, drafts, vocab]")
    if counts is not None and tuple(counts.shape) != (n,):
        raise ValueError("counts must be [n]")
    device = target_probs.device
    given = [draft_tokens, uniforms, noise] + [t for t in (draft_probs, counts) if t is not None]
    if device.type != "cuda" or any(t.device != device for t in given):
        raise RuntimeError("verification tensors must share a CUDA device")
    if target_probs.dtype not in _lib.DTYPE_CODES or (draft_probs is not None
                                                      and draft_probs.dtype != target_probs.dtype):
        raise RuntimeError("probabilities must share an fp32/fp16/bf16 dtype")
    if draft_tokens.dtype != torch.int64 or uniforms.dtype != torch.float32 or noise.dtype != torch.float32:
        raise RuntimeError("draft_tokens must be int64, uniforms and noise fp32")
    if counts is not None and counts.dtype != torch.int32:
        raise RuntimeError("counts must be int32")
    target_probs = target_probs if target_probs.stride(2) == 1 else target_probs.contiguous()
    if draft_probs is not None and draft_probs.stride(2) != 1:
        draft_probs = draft_probs.contiguous()
    draft_tokens, uniforms, noise = draft_tokens.contiguous(), uniforms.contiguous(), noise.contiguous()
    counts = None if counts is None else counts.contiguous()
    tokens = torch.empty((n, drafts + 1), dtype=torch.int64, device=device)
    accepted = torch.empty(n, dtype=torch.int32, device=device)
    args = (target_probs.data_ptr(), target_probs.stride(0), target_probs.stride(1),
            None if draft_probs is None else draft_probs.data_ptr(),
            0 if draft_probs is None else draft_probs.stride(0), 0 if draft_probs is None else draft_probs.stride(1),
            _lib.DTYPE_CODES[target_probs.dtype], n, drafts, vocab, draft_tokens.data_ptr(),
            None if counts is None else counts.data_ptr(), uniforms.data_ptr(), noise.data_ptr(), tokens.data_ptr(),
            accepted.data_ptr())
    with torch.cuda.device(device):
        _lib.check(_lib.lib().popkv_verify_drafts(*args, torch.cuda.current_stream(device).cuda_stream))
    return tokens, accepted
