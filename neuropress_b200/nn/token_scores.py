"""Scoring given tokens with a (lowered) lm_head: log probabilities, entropy, top alternatives.

The measure of what a compressed model lost -- perplexity, token-level divergence -- needs the log
probability of given tokens at many positions.  The logits of a long text are a [positions,
vocabulary] matrix that nobody else reads: :func:`score_tokens` runs the lm_head over chunks of
positions and ``kernels.token_logprobs`` over each chunk's logits, so only one chunk of them exists
at a time.  No reference counterpart (the reference leaves this to an external harness).
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

__all__ = ["TokenScores", "score_tokens"]


class TokenScores(NamedTuple):
    logprob: torch.Tensor        # fp32 [...], 0 where the target is outside the vocabulary
    entropy: torch.Tensor        # fp32 [...], nats
    top_logprobs: torch.Tensor   # fp32 [..., top_n]
    top_ids: torch.Tensor        # int64 [..., top_n]


def score_tokens(lm_head: nn.Module, hidden: torch.Tensor, targets: torch.Tensor, top_n: int = 0,
                 rows_per_chunk: int = 1024, vocab_size: int | None = None) -> TokenScores:
    """``hidden`` ``[..., H]`` are the states that predict ``targets`` ``[...]`` (int64; an id outside the vocabulary,
    such as an ignore index, scores 0).  ``vocab_size`` cuts the logits of a padded lm_head, which must have that many."""
    from .. import kernels

    if hidden.dim() < 1 or hidden.shape[:-1] != targets.shape:
        raise RuntimeError("score_tokens: expected hidden [..., H] and targets [...].")
    if rows_per_chunk < 1:
        raise RuntimeError("score_tokens: rows_per_chunk must be positive.")
    if vocab_size is not None and vocab_size < 1:
        raise RuntimeError("score_tokens: vocab_size must be positive.")
    leading, rows = targets.shape, targets.numel()
    h2, t2 = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1).contiguous()
    if rows == 0:
        empty = hidden.new_empty(leading, dtype=torch.float32)
        return TokenScores(empty, empty.clone(), hidden.new_empty((*leading, top_n), dtype=torch.float32),
                           targets.new_empty((*leading, top_n)))
    parts = []
    for r in range(0, rows, rows_per_chunk):
        logits = lm_head(h2[r:r + rows_per_chunk])
        if vocab_size is not None:
            if vocab_size > logits.shape[-1]:
                raise RuntimeError(f"score_tokens: vocab_size is {vocab_size}, the lm_head has {logits.shape[-1]} logits.")
            logits = logits[:, :vocab_size]
        parts.append(kernels.token_logprobs(logits, t2[r:r + rows_per_chunk], top_n=top_n))
    whole = parts[0] if len(parts) == 1 else [torch.cat(p) for p in zip(*parts)]
    return TokenScores(*(w.reshape(*leading, *w.shape[1:]) for w in whole))
