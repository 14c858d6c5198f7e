"""Verification of drafted tokens (speculative sampling) from given random numbers."""

from __future__ import annotations

import torch

from . import _lib


def verify_drafts(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, draft_tokens: torch.Tensor,
                  uniform: torch.Tensor, noise: torch.Tensor, *, draft_counts: torch.Tensor | None = None,
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Accept drafts while ``uniform * q < p`` and draw the next token
    (tq_verify_drafts).

    ``target_probs`` ``[seqs, drafts + 1, vocab]`` and ``draft_probs`` ``[seqs,
    drafts, vocab]`` (fp32, fp16 or bf16; ``None`` for a drafter that was
    certain of its tokens), ``draft_tokens`` int32 ``[seqs, drafts]``,
    ``uniform`` fp32 ``[seqs, drafts]`` in [0, 1), ``noise`` fp32 ``[seqs,
    vocab]`` of unit-exponential numbers, ``draft_counts`` int32 ``[seqs]`` where
    sequences have fewer drafts than ``drafts``.

    Returns ``(accepted [seqs], tokens [seqs, drafts + 1])``, both int32: the
    accepted drafts, then the next token - drawn from the normalised
    ``max(p - q, 0)`` at the first rejection, or from ``p`` after the last draft
    - then -1s.  The draw is ``argmax(weight / noise)``, ties to the lowest
    token, so the same numbers give the same tokens on every run."""
    lib = _lib.load()
    index = target_probs.get_device()
    seqs, rows, vocab = target_probs.shape if target_probs.dim() == 3 else (0, 0, 0)
    if rows < 1 or vocab < 1 or index < 0:
        raise ValueError("target_probs must be a CUDA tensor [seqs, drafts + 1, vocab]")
    if _lib.current_device() != index:
        with torch.cuda.device(index):
            return verify_drafts(target_probs, draft_probs, draft_tokens, uniform, noise, draft_counts=draft_counts)
    dev, drafts, dtype = target_probs.device, rows - 1, target_probs.dtype
    code = _lib.dtype_code(dtype)
    target_seq, target_row, inner = target_probs.stride()
    if inner != 1 and vocab > 1:
        target_probs = target_probs.contiguous()
        target_seq, target_row, _ = target_probs.stride()
    draft, draft_seq, draft_row = None, 0, 0
    if draft_probs is not None:
        if draft_probs.shape != (seqs, drafts, vocab) or draft_probs.dtype is not dtype \
                or draft_probs.get_device() != index:
            raise ValueError(f"draft_probs must be {dtype} [{seqs}, {drafts}, {vocab}] on {dev}")
        draft_seq, draft_row, inner = draft_probs.stride()
        if inner != 1 and vocab > 1:
            draft_probs = draft_probs.contiguous()
            draft_seq, draft_row, _ = draft_probs.stride()
        draft = draft_probs.data_ptr()
    if draft_tokens.dtype is not torch.int32 or draft_tokens.shape != (seqs, drafts) \
            or draft_tokens.get_device() != index:
        raise ValueError(f"draft_tokens must be int32 [{seqs}, {drafts}] on {dev}")
    if uniform.dtype is not torch.float32 or uniform.shape != (seqs, drafts) or uniform.get_device() != index:
        raise ValueError(f"uniform must be fp32 [{seqs}, {drafts}] on {dev}")
    if noise.dtype is not torch.float32 or noise.shape != (seqs, vocab) or noise.get_device() != index:
        raise ValueError(f"noise must be fp32 [{seqs}, {vocab}] on {dev}")
    counts = None
    if draft_counts is not None:
        if (draft_counts.dtype is not torch.int32 or draft_counts.shape != (seqs,) or draft_counts.get_device() != index
                or not draft_counts.is_contiguous()):
            raise ValueError(f"draft_counts must be contiguous int32 [{seqs}] on {dev}")
        counts = draft_counts.data_ptr()
    if not draft_tokens.is_contiguous():
        draft_tokens = draft_tokens.contiguous()
    if not uniform.is_contiguous():
        uniform = uniform.contiguous()
    if noise.stride(1) != 1 and vocab > 1:
        noise = noise.contiguous()
    accepted = draft_tokens.new_empty((seqs,))
    tokens = draft_tokens.new_empty((seqs, rows))
    status = lib.tq_verify_drafts(target_probs.data_ptr(), target_seq, target_row, draft, draft_seq, draft_row, code,
                                  draft_tokens.data_ptr(), counts, uniform.data_ptr(), noise.data_ptr(),
                                  noise.stride(0), seqs, drafts, vocab, accepted.data_ptr(), tokens.data_ptr(),
                                  _lib.stream_of(index))
    if status:
        _lib.check(status, "verify drafts")
    return accepted, tokens
