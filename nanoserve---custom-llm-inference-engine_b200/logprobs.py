"""Log-probabilities of sampled or given tokens, their ranks, and each row's
most likely tokens: what a serving API returns next to the ids of a step
(``logprobs`` / ``top_logprobs``) or for the tokens of a prompt.  No
counterpart in the reference.  Serving only: there is no gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _cabi
from .sampler import _Op

_token_logprobs = _Op("token_logprobs")

MAX_TOP = _cabi.NS_MAX_TOP_LOGPROBS


class TokenLogprobs(NamedTuple):
    """One row per token."""

    logprobs: torch.Tensor      # float32 [S]         log-probability of the row's token
    ranks: torch.Tensor         # int32 [S]           1 + how many tokens are more likely
    top_ids: torch.Tensor       # like token_ids [S, top_n]  the most likely tokens, best first
    top_logprobs: torch.Tensor  # float32 [S, top_n]  their log-probabilities


def token_logprobs(
    logits: torch.Tensor,
    token_ids: torch.Tensor,
    top_n: int = 0,
    *,
    sample_indices: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> TokenLogprobs:
    """``log_softmax(logits[i])[token_ids[i]]`` for every row ``i``, its rank, and the
    ``top_n`` (at most 32) most likely tokens.

    ``logits`` is fp32 or bf16 ``[T, V]``; row ``i`` reads ``logits[sample_indices[i]]``
    (or ``logits[i]``).  ``token_ids`` is int64 or int32 ``[S]``.  Equal logits
    rank by ascending id among the top tokens and share the better
    ``ranks``.  A row that the sampler's guard makes uniform (a NaN, a +inf or
    only -inf, nanoserve/scheduler/sampler.py:78-80) has log-probability
    ``-log(V)`` everywhere, rank 1 and ``top_ids`` ``0 .. top_n-1``.  A token id
    outside ``[0, V)`` gets NaN and rank 0, and sets ``NS_STATUS_BAD_TOKEN_ID`` in
    ``status`` (int32 ``[1]``).  One launch on the current stream of
    ``logits.device``; no synchronisation, graph-capturable."""
    return TokenLogprobs(*_token_logprobs(logits, sample_indices, token_ids, top_n, status))
