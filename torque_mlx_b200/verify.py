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
    return _lib.binding().verify_drafts(target_probs, draft_probs, draft_tokens, uniform, noise, draft_counts)
