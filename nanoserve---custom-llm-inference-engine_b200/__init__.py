"""B200-native (sm_100a) replacement for NanoServe's token-sampling hot path.

Public surface:

* :class:`Sampler` -- drop-in for ``nanoserve.scheduler.sampler.Sampler``
  (nanoserve/scheduler/sampler.py:17-89), backed by
  ``torch.ops.nanoserve_b200.sample``;
* :class:`SamplingParams` -- same fields as nanoserve/config.py:68-79, and
  :class:`ExtendedSamplingParams` -- with presence and frequency penalties and
  a ``logit_bias``;
* :func:`process_logits` -- penalties, biases and grammar masks on logits;
* :func:`token_logprobs` -- log-probabilities, ranks and most likely tokens;
* :mod:`._cabi` -- ctypes binding of ``include/nanoserve_sampler.h``;
* :class:`HistoryStore` -- device-resident, append-only prior-token
  histories (replaces the per-step lists of nanoserve/engine.py:242-246);
* :class:`PagedHistoryStore` -- the same in pages that forks of a request
  share, with :class:`PageAllocator`, :func:`copy_pages` and
  :func:`gather_paged_history` (which serve any paged cache);
* :mod:`.sharded` -- row-sharded sampling over several GPUs (one process per
  GPU, one NCCL all-gather of the sampled ids);
* :mod:`.workloads` -- seeded synthetic inputs shaped like the benchmark
  configurations.
"""
from .config import ExtendedSamplingParams, SamplingParams
from .sampler import Sampler, load_ops
from .history import HistoryStore
from .logits import process_logits
from .logprobs import TokenLogprobs, token_logprobs
from .pages import PageAllocator, PagedHistoryStore, copy_pages, gather_paged_history

__all__ = [
    "ExtendedSamplingParams", "HistoryStore", "PageAllocator", "PagedHistoryStore", "Sampler", "SamplingParams",
    "TokenLogprobs", "copy_pages", "gather_paged_history", "load_ops", "process_logits", "token_logprobs",
]
