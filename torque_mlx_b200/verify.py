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
    if target_probs.dim() != 3 or not target_probs.is_cuda or target_probs.shape[1] < 1:
        raise ValueError("target_probs must be a CUDA tensor [seqs, drafts + 1, vocab]")
    dev = target_probs.device
    seqs, rows, vocab = target_probs.shape
    drafts = rows - 1
    code = _lib.dtype_code(target_probs.dtype)
    if vocab < 1:
        raise ValueError("the vocabulary is empty")
    if target_probs.stride(2) != 1 and vocab > 1:
        target_probs = target_probs.contiguous()
    dp, dss, dsr = None, 0, 0
    if draft_probs is not None:
        if tuple(draft_probs.shape) != (seqs, drafts, vocab) or draft_probs.dtype != target_probs.dtype \
                or draft_probs.device != dev:
            raise ValueError(f"draft_probs must be {target_probs.dtype} [{seqs}, {drafts}, {vocab}] on {dev}")
        if draft_probs.stride(2) != 1 and vocab > 1:
            draft_probs = draft_probs.contiguous()
        dp, dss, dsr = draft_probs.data_ptr(), draft_probs.stride(0), draft_probs.stride(1)
    if draft_tokens.dtype != torch.int32 or tuple(draft_tokens.shape) != (seqs, drafts) or draft_tokens.device != dev:
        raise ValueError(f"draft_tokens must be int32 [{seqs}, {drafts}] on {dev}")
    if uniform.dtype != torch.float32 or tuple(uniform.shape) != (seqs, drafts) or uniform.device != dev:
        raise ValueError(f"uniform must be fp32 [{seqs}, {drafts}] on {dev}")
    if noise.dtype != torch.float32 or tuple(noise.shape) != (seqs, vocab) or noise.device != dev:
        raise ValueError(f"noise must be fp32 [{seqs}, {vocab}] on {dev}")
    counts = None
    if draft_counts is not None:
        if (draft_counts.dtype != torch.int32 or tuple(draft_counts.shape) != (seqs,) or draft_counts.device != dev
                or not draft_counts.is_contiguous()):
            raise ValueError(f"draft_counts must be contiguous int32 [{seqs}] on {dev}")
        counts = draft_counts.data_ptr()
    draft_tokens, uniform = draft_tokens.contiguous(), uniform.contiguous()
    if noise.stride(1) != 1 and vocab > 1:
        noise = noise.contiguous()
    accepted = torch.empty((seqs,), dtype=torch.int32, device=dev)
    tokens = torch.empty((seqs, rows), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.tq_verify_drafts(
            target_probs.data_ptr(), target_probs.stride(0), target_probs.stride(1), dp, dss, dsr, code,
            draft_tokens.data_ptr(), counts, uniform.data_ptr(), noise.data_ptr(), noise.stride(0), seqs, drafts, vocab,
            accepted.data_ptr(), tokens.data_ptr(), _lib.stream_ptr()), "verify drafts")
    return accepted, tokens
