"""Verification of drafted tokens (speculative decoding).

``verify_drafts`` decides, on the device and without a host round trip, how many of each
sequence's drafted tokens the target model keeps and which token follows them.  The accepted
tokens and the following one are distributed exactly as the target's own samples.

The reference decodes one token per call (popkv.py:988-1115) and has no counterpart.
"""
from __future__ import annotations

import struct

import torch

from . import _lib

_WORDS = struct.Struct("18q").pack  # see popkv_verify_drafts_words


_workspaces: dict[tuple[int, int], torch.Tensor] = {}  # of each (device, stream): all zero between calls


def verify_workspace(n: int, device) -> torch.Tensor:
    """Scratch for ``verify_drafts`` calls of up to ``n`` sequences, zeroed.

    Without one, calls keep one per stream; inside a graph capture each call would make and clear its
    own.  Calls that overlap in time need one each.
    """
    return torch.zeros(12 * n, dtype=torch.uint8, device=device)


def _workspace(given, n: int, device, stream: int) -> torch.Tensor:
    if given is not None:
        if given.dtype != torch.uint8 or not given.is_contiguous() or given.device != device or given.numel() < 12 * n:
            raise ValueError(f"workspace must be a tensor of verify_workspace({n}, ...)")
        return given
    if torch.cuda.is_current_stream_capturing():
        return verify_workspace(n, device)
    held = _workspaces.get((device.index, stream))
    if held is None or held.shape[0] < 12 * n:
        held = _workspaces[device.index, stream] = verify_workspace(n, device)
    return held


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                  noise: torch.Tensor, *, draft_probs: torch.Tensor | None = None,
                  counts: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
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
        workspace: a tensor of ``verify_workspace``, for calls inside a graph capture.

    Draft j is accepted while ``uniforms * q(draft) < p(draft)``.  The following token wins the race
    ``argmax weight / noise`` over weight > 0, weight = max(p - q, 0) at the first refusal (p where
    that is zero everywhere) and p after the last draft; ties go to the lowest id.

    Returns (tokens int64 [n, drafts + 1]: accepted drafts, the following token, then -1; accepted
    int32 [n]).
    """
    if target_probs.ndim != 3 or draft_tokens.ndim != 2:
        raise ValueError("target_probs must be [n, drafts + 1, vocab] and draft_tokens [n, drafts]")
    n, drafts = draft_tokens.shape
    shape = target_probs.shape
    vocab = shape[2]
    if shape[0] != n or shape[1] != drafts + 1 or vocab < 1:
        raise ValueError("target_probs must be [n, drafts + 1, vocab]")
    if uniforms.shape != (n, drafts) or noise.shape != (n, vocab):
        raise ValueError("uniforms must be [n, drafts] and noise [n, vocab]")
    dtype, device = target_probs.dtype, target_probs.device
    together = device.type == "cuda" and draft_tokens.device == uniforms.device == noise.device == device
    code = _lib.DTYPE_CODES.get(dtype)
    typed = code is not None
    if draft_probs is not None:
        if draft_probs.shape != (n, drafts, vocab):
            raise ValueError("draft_probs must be [n, drafts, vocab]")
        together = together and draft_probs.device == device
        typed = typed and draft_probs.dtype == dtype
    if counts is not None:
        if counts.shape != (n,):
            raise ValueError("counts must be [n]")
        together = together and counts.device == device
    if not together:
        raise RuntimeError("verification tensors must share a CUDA device")
    if not typed:
        raise RuntimeError("probabilities must share an fp32/fp16/bf16 dtype")
    if draft_tokens.dtype != torch.int64 or uniforms.dtype != torch.float32 or noise.dtype != torch.float32:
        raise RuntimeError("draft_tokens must be int64, uniforms and noise fp32")
    if counts is not None and counts.dtype != torch.int32:
        raise RuntimeError("counts must be int32")
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _verify(target_probs, draft_tokens, uniforms, noise, draft_probs, counts, workspace, code)
    return _verify(target_probs, draft_tokens, uniforms, noise, draft_probs, counts, workspace, code)


def _verify(target_probs, draft_tokens, uniforms, noise, draft_probs, counts, workspace, code):
    n, places, vocab = target_probs.shape
    device = target_probs.device
    target_probs = target_probs if target_probs.stride(2) == 1 else target_probs.contiguous()
    draft, d_seq, d_place = 0, 0, 0
    if draft_probs is not None:
        draft_probs = draft_probs if draft_probs.stride(2) == 1 else draft_probs.contiguous()
        draft, (d_seq, d_place, _) = draft_probs.data_ptr(), draft_probs.stride()
    draft_tokens, uniforms, noise = draft_tokens.contiguous(), uniforms.contiguous(), noise.contiguous()
    counts = None if counts is None else counts.contiguous()
    tokens, accepted = draft_tokens.new_empty((n, places)), draft_tokens.new_empty(n, dtype=torch.int32)
    stream = _lib.raw_stream(device.index)
    scratch = _workspace(workspace, n, device, stream)
    t_seq, t_place, _ = target_probs.stride()
    status = _lib.lib().popkv_verify_drafts_words(_WORDS(
        target_probs.data_ptr(), t_seq, t_place, draft, d_seq, d_place, code, n, places - 1, vocab,
        draft_tokens.data_ptr(), 0 if counts is None else counts.data_ptr(), uniforms.data_ptr(),
        noise.data_ptr(), scratch.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), stream))
    if status:
        _lib.check(status)
    return tokens, accepted
