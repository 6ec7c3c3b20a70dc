"""Penalties for repeated tokens, biases and grammar masks on logits.

The reference knows one penalty (nanoserve/scheduler/sampler.py:31-38).  A
serving API asks for more: presence and frequency penalties on the generated
tokens, a ``logit_bias`` per request, and masks of the tokens that a grammar
allows next.  ``process_logits`` applies all of them in one launch
(``ns_process_logits``); ``Sampler.sample`` and the history stores call it for
requests that carry such fields.  Serving only: there is no gradient.
"""
from __future__ import annotations

from typing import Optional

import torch

from .sampler import _Op

_process = _Op("process_logits")
_process_into = _Op("process_logits_")


def process_logits(
    logits: torch.Tensor,
    *,
    sample_indices: Optional[torch.Tensor] = None,
    history_offsets: Optional[torch.Tensor] = None,
    history_ids: Optional[torch.Tensor] = None,
    prompt_lens: Optional[torch.Tensor] = None,
    repetition_penalty: Optional[torch.Tensor] = None,
    presence_penalty: Optional[torch.Tensor] = None,
    frequency_penalty: Optional[torch.Tensor] = None,
    bias_offsets: Optional[torch.Tensor] = None,
    bias_ids: Optional[torch.Tensor] = None,
    bias_values: Optional[torch.Tensor] = None,
    allowed: Optional[torch.Tensor] = None,
    allowed_rows: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Processed logits ``[S, V]`` of ``S`` rows.

    Row ``i`` reads ``logits[sample_indices[i]]`` (or ``logits[i]``), fp32 or
    bf16.  With its history ``history_ids[history_offsets[i]:history_offsets[i+1]]``
    and, for a token ``v``, ``seen`` = it occurs there and ``c`` = how often it
    occurs from position ``prompt_lens[i]`` on (default 0: all of it)::

        x = x * rp if x < 0 else x / rp      where seen
        x = x - frequency * c - presence     where c > 0
        x = x + bias                         where the row has one for v
        x = -inf                             where the row's mask forbids v

    computed in fp32 and rounded once to ``out``'s type.  All arguments are
    device tensors on ``logits.device``; what is not given is not applied:

    * ``history_offsets`` int64 ``[S+1]``, ``history_ids`` int32,
      ``prompt_lens`` int32 ``[S]``;
    * ``repetition_penalty``, ``presence_penalty``, ``frequency_penalty``
      float32 ``[S]``;
    * ``bias_offsets`` int64 ``[S+1]``, ``bias_ids`` int32, ``bias_values``
      float32, at most 2^18 a row (a longer list is left out, as a bad range): if
      a row names an id twice, its last entry counts;
    * ``allowed`` int32 ``[M, >= ceil(V/32)]``: token ``v`` is allowed where bit
      ``v % 32`` of word ``v // 32`` is 1.  ``allowed_rows`` int32 ``[S]`` gives
      each row's mask, a negative one none; without it row ``i`` has mask
      ``i``.  A row whose mask allows nothing becomes all ``-inf``, which the
      sampler treats as uniform (nanoserve/scheduler/sampler.py:78-80).

    ``out`` may be ``logits`` itself: then only what changes is written.
    Otherwise it must not overlap them, and ``logits`` is left as it was.
    An ``out`` that requires a gradient is refused while gradients are enabled.
    ``out_dtype`` (when ``out`` is not given) is the logits' type or float32.
    Bad ids, ranges and indices are skipped and set ``NS_STATUS_*`` bits in
    ``status`` (int32 ``[1]``).  One launch on the current stream of
    ``logits.device``; no synchronisation, graph-capturable."""
    if out is None:
        return _process(logits, sample_indices, history_offsets, history_ids, prompt_lens, repetition_penalty,
                        presence_penalty, frequency_penalty, bias_offsets, bias_ids, bias_values, allowed,
                        allowed_rows, status, out_dtype)
    if out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out has dtype {out.dtype}, out_dtype is {out_dtype}")
    if out is not logits and logits.dim() == 2 and logits.shape[1] > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    _process_into(logits, sample_indices, history_offsets, history_ids, prompt_lens, repetition_penalty,
                  presence_penalty, frequency_penalty, bias_offsets, bias_ids, bias_values, allowed, allowed_rows,
                  status, out)
    return out
