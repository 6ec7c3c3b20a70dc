"""Drop-in replacement for nanoserve/scheduler/sampler.py (``Sampler``).

``Sampler(device).sample(logits, sampling_params_list, history_token_ids,
generators=None)`` keeps the reference signature (sampler.py:17-27) and
returns int64 token ids on ``logits.device``, so ``engine.py:247-250`` and
``Scheduler.update_with_sampled`` work unchanged.  The work is one call of
the sm_100a library behind ``torch.ops.nanoserve_b200.sample``: one kernel
launch, enqueued on the current stream of ``logits.device``.  The call is
wrapped in an NVTX range named ``logits+sample``, the range the reference's
engine opens around the same step (nanoserve/engine/engine.py:234).

Differences from the reference, all additive:

* the input ``logits`` is never modified (the reference writes the penalised
  logits back into it, sampler.py:38; ``return_debug=True`` returns them);
* keyword-only extensions: ``sample_indices`` (fused row gather from a flat
  ``[T, V]`` fp32/bf16 tensor), ``uniforms`` (one caller uniform per row),
  ``seed`` (Philox key), ``out_dtype`` (int64 or int32);
* randomness comes from per-row Philox4x32-10 streams keyed by
  ``(seed, step, row)`` instead of the global generator that
  ``torch.multinomial`` uses (sampler.py:87); ``SamplingParams.seed``, which
  the reference ignores, gives a request its own stream, keyed by the seed
  and the length of its history, so it draws the same tokens whatever batch
  it is in;
* requests may carry presence and frequency penalties and a ``logit_bias``
  (``ExtendedSamplingParams``), and ``allowed`` masks the tokens that a grammar
  allows; ``logprobs=n`` also returns the log-probabilities of the sampled
  tokens and of the ``n`` most likely ones;
* ``generators`` is accepted and ignored, as in the reference (sampler.py:26);
* ``sample_async`` returns int32 ids through a non-blocking copy to pinned
  host memory (``PendingTokens.wait()``), in place of the caller's blocking
  ``.tolist()`` (engine.py:250).

There is no CPU path: the op raises if the CUDA library is not built or the
tensors are not on a CUDA device.
"""
from __future__ import annotations

from pathlib import Path
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import packing

_PKG_DIR = Path(__file__).resolve().parent
_OPS_PATH = _PKG_DIR / "_nanoserve_ops.so"
_ops_loaded = False


def load_ops() -> None:
    """Register torch.ops.nanoserve_b200.* (raises if the library was not built)."""
    global _ops_loaded
    if _ops_loaded:
        return
    if not _OPS_PATH.exists():
        raise RuntimeError(
            f"{_OPS_PATH} is missing: build it with __graft_entry__.build() "
            "(there is no CPU fallback for the sampling op)"
        )
    torch.ops.load_library(str(_OPS_PATH))
    _ops_loaded = True


class _Op:
    """``torch.ops.nanoserve_b200.<name>``, looked up at its first call."""

    def __init__(self, name: str):
        self._name = name
        self._op = None

    def __call__(self, *args):
        if self._op is None:
            load_ops()
            self._op = getattr(torch.ops.nanoserve_b200, self._name).default
        return self._op(*args)


class _Staging:
    """A reusable pinned host buffer plus the event of its last H2D copy."""

    def __init__(self) -> None:
        self.host: Optional[torch.Tensor] = None
        self.event: Optional[torch.cuda.Event] = None

    def get(self, nbytes: int) -> torch.Tensor:
        if self.event is not None:
            self.event.synchronize()
        if self.host is None or self.host.numel() < nbytes:
            cap = max(nbytes, 1 << 16)
            self.host = torch.empty(cap, dtype=torch.uint8, pin_memory=True)
        return self.host[:nbytes]


class PendingTokens:
    """Sampled ids on their way to the host: an int32 copy into pinned memory,
    enqueued behind the sampling kernel, and the event that marks its end.
    ``wait()`` blocks until then and returns the ids as a list (what
    ``engine.py:250`` gets from ``.tolist()``)."""

    def __init__(self, host: torch.Tensor, event: torch.cuda.Event, n: int):
        self._host = host
        self._event = event
        self._n = n
        self._ids: Optional[List[int]] = None

    def ready(self) -> bool:
        return self._ids is not None or self._event.query()

    def wait(self) -> List[int]:
        if self._ids is None:
            self._event.synchronize()
            self._ids = self._host[: self._n].numpy().tolist()
        return self._ids


class _HostRing:
    """A few pinned int32 buffers reused round robin for PendingTokens; a
    buffer is handed out again only after its previous copy has finished."""

    def __init__(self, slots: int = 4):
        self._bufs: List[Optional[torch.Tensor]] = [None] * slots
        self._pending: List[Optional[PendingTokens]] = [None] * slots
        self._next = 0

    def copy(self, tokens: torch.Tensor) -> PendingTokens:
        i = self._next
        self._next = (i + 1) % len(self._bufs)
        prev = self._pending[i]
        if prev is not None:
            prev.wait()  # its list is taken before the buffer is reused
        n = tokens.numel()
        if self._bufs[i] is None or self._bufs[i].numel() < n:
            self._bufs[i] = torch.empty(max(n, 1024), dtype=torch.int32, pin_memory=True)
        host = self._bufs[i]
        src = tokens if tokens.dtype == torch.int32 else tokens.to(torch.int32)
        with torch.cuda.device(tokens.device):
            host[:n].copy_(src, non_blocking=True)
            ev = torch.cuda.Event()
            ev.record(torch.cuda.current_stream(tokens.device))
        pt = PendingTokens(host, ev, n)
        self._pending[i] = pt
        return pt


KERNELS = {"auto": 0, "cluster": 1, "split": 2}


class Sampler:
    """B200 sampling op with the reference ``Sampler`` interface.

    ``kernel`` picks the CUDA kernel: ``"auto"`` (the row kernel, whose
    persistent blocks split the batch's rows among the SMs, for
    batches of at least 32 aligned rows, the cluster kernel otherwise),
    ``"cluster"`` or ``"split"`` (where its layout conditions hold)."""

    def __init__(self, device, kernel: str = "auto"):
        if kernel not in KERNELS:
            raise ValueError(f"kernel must be one of {sorted(KERNELS)}")
        self.device = torch.device(device)
        self.kernel = kernel
        self._step = 0
        self._staging = _Staging()
        self._ring = _HostRing()
        load_ops()

    def sample_async(self, logits: torch.Tensor, sampling_params_list: List,
                     history_token_ids: List[List[int]], generators=None, **kw) -> PendingTokens:
        """``sample`` with int32 ids and a non-blocking copy to pinned host
        memory in place of the caller's blocking ``.tolist()`` (engine.py:250):
        the host can prepare the next step while this one samples, then
        ``wait()``.  Up to four results may be outstanding at once; a fifth
        call first waits for the oldest."""
        if kw.get("return_debug"):
            raise ValueError("sample_async returns ids only; use sample(return_debug=True) for debug outputs")
        if kw.get("logprobs") is not None:
            raise ValueError("sample_async returns ids only; use sample(logprobs=n) for log-probabilities")
        kw["out_dtype"] = torch.int32
        out = self.sample(logits, sampling_params_list, history_token_ids, generators, **kw)
        return self._ring.copy(out)

    def to_host_async(self, tokens: torch.Tensor) -> PendingTokens:
        """Non-blocking int32 copy of device ids (e.g. from ``sample_packed`` or
        ``HistoryStore.sample``) to pinned host memory."""
        return self._ring.copy(tokens)

    # -- the reference entry point (sampler.py:21-27) ---------------------
    def sample(
        self,
        logits: torch.Tensor,
        sampling_params_list: List,
        history_token_ids: List[List[int]],
        generators: Optional[List[Optional[torch.Generator]]] = None,
        *,
        sample_indices: Optional[torch.Tensor] = None,
        uniforms: Optional[torch.Tensor] = None,
        seed: Optional[int] = None,
        out_dtype: torch.dtype = torch.int64,
        return_debug: bool = False,
        prompt_lens: Optional[Sequence[int]] = None,
        allowed: Optional[torch.Tensor] = None,
        allowed_rows: Optional[torch.Tensor] = None,
        logprobs: Optional[int] = None,
    ):
        """The next token of every row.

        Rows whose parameters carry presence or frequency penalties or a
        ``logit_bias`` (``ExtendedSamplingParams``), or any row when ``allowed`` is
        given, are first processed by :func:`process_logits` (into a copy;
        ``prompt_lens[i]`` ids of row i's history are its prompt, ``allowed`` and
        ``allowed_rows`` are that function's device tensors).  With ``logprobs=n``
        the result is ``(result, TokenLogprobs)``: the log-probabilities, over the
        logits after all penalties (the repetition penalty among them), biases
        and masks and before temperature and filters, of the sampled tokens
        and of the ``n`` most likely ones.

        A row that has nothing left to draw (its mask allows no token, the logits or
        biases of those it allows are all -inf, or one of them is NaN or +inf) is
        drawn uniformly from the whole vocabulary, as the reference draws such rows
        (nanoserve/scheduler/sampler.py:78-80), forbidden tokens included; a greedy
        one gets token 0, or the first NaN or +inf.  Its
        log-probabilities are ``-log(V)`` and its rank is 1: a caller that cannot
        rule such rows out asks for ``logprobs=0`` and looks."""
        if logits.dim() != 2:
            raise ValueError("logits must be [num_seqs, vocab]")
        if not logits.is_cuda:
            raise RuntimeError("Sampler.sample needs CUDA logits (no CPU fallback)")
        if allowed_rows is not None and allowed is None:
            raise ValueError("allowed_rows given without allowed")
        vocab = logits.shape[1]
        S = len(sampling_params_list)
        if sample_indices is None and logits.shape[0] != S:
            raise ValueError(f"logits has {logits.shape[0]} rows but {S} sampling params were given")
        torch.cuda.nvtx.range_push("logits+sample")
        try:
            # every copy, event and launch below goes to the logits' device,
            # whatever device is current for the caller
            with torch.cuda.device(logits.device):
                step = dict(uniforms=uniforms, seed=seed, out_dtype=out_dtype, return_debug=return_debug)
                if allowed is not None or packing.wants_processing(sampling_params_list):
                    return self._sample_processed(
                        logits, sampling_params_list, _ListHistories(history_token_ids, S, vocab), prompt_lens,
                        sample_indices=sample_indices, allowed=allowed, allowed_rows=allowed_rows, logprobs=logprobs,
                        **step,
                    )
                packed = packing.pack_plain(sampling_params_list, history_token_ids, vocab,
                                            sms=_sm_count(logits.device))
                row_params, offsets, ids, order = self._upload(packed, logits.device)
                out = self.sample_packed(
                    logits, row_params, offsets, ids, sample_indices=sample_indices, row_order=order, **step,
                )
                return self._with_logprobs(out, logits, logprobs, sample_indices, row_params, offsets, ids)
        finally:
            torch.cuda.nvtx.range_pop()

    def _sample_processed(self, logits: torch.Tensor, params: Sequence, histories, prompt_lens, *,
                          sample_indices: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                          allowed_rows: Optional[torch.Tensor] = None, logprobs: Optional[int] = None, **step):
        """``sample`` with the logits processed first (penalties, the
        repetition penalty among them, biases and masks), into an fp32 copy of
        the sampled rows.  ``histories`` gives the lengths of the rows'
        histories, the host arrays to upload for the ids of the rows that need
        them, and those ids on the device.  With ``return_debug`` the status holds
        what the processing reports too (bad sample indices, ids and masks)."""
        from .logits import process_logits

        dev, vocab = logits.device, logits.shape[1]
        if sample_indices is None and logits.shape[0] != len(params):
            raise ValueError(f"logits has {logits.shape[0]} rows but {len(params)} sampling params were given")
        lens = histories.lens()
        pr = packing.pack_processing(params, lens, prompt_lens, vocab)
        rows = packing.derive_rows(params, vocab, lens)
        rows["flags"] &= ~np.uint32(packing._cabi.NS_ROW_PENALTY)  # applied here
        order = packing.schedule(rows, _sm_count(dev))
        # what no row uses is neither uploaded nor applied
        total = int(pr.offsets[-1])
        parts = {"rows": rows.view(np.uint8), "order": order}
        if total:
            parts.update(history_offsets=pr.offsets, repetition_penalty=pr.repetition,
                         presence_penalty=pr.presence, frequency_penalty=pr.frequency)
            if prompt_lens is not None:
                parts["prompt_lens"] = pr.prompt_lens
        if pr.bias_ids.size:
            parts.update(bias_offsets=pr.bias_offsets, bias_ids=pr.bias_ids, bias_values=pr.bias_values)
        more = histories.parts(pr.lens) if total else []
        up = upload_parts(self._staging, [*parts.values(), *more], dev)
        given = dict(zip(parts, up))
        row_params, order_d = given.pop("rows"), given.pop("order")
        if total:
            given["history_ids"] = histories.ids(up[len(parts):], given["history_offsets"], total)
        status = torch.zeros(1, dtype=torch.int32, device=dev) if step.get("return_debug") else None
        processed = process_logits(logits.detach(), sample_indices=sample_indices, allowed=allowed,
                                   allowed_rows=allowed_rows, out_dtype=torch.float32, status=status, **given)
        out = self.sample_packed(processed, row_params, None, None, row_order=order_d, **step)
        if status is not None:
            out[1]["status"].bitwise_or_(status)
        return self._with_logprobs(out, processed, logprobs, None)

    @staticmethod
    def _with_logprobs(out, logits: torch.Tensor, logprobs: Optional[int], sample_indices: Optional[torch.Tensor],
                       row_params: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                       ids: Optional[torch.Tensor] = None):
        """``out``, and the log-probabilities of its tokens if they are asked for.  Histories (of the rows that the
        sampler penalised itself, in ``row_params``) say that an fp32 copy is penalised first, as the sampler does."""
        if logprobs is None:
            return out
        from .logits import process_logits
        from .logprobs import token_logprobs

        tokens = out[0] if isinstance(out, tuple) else out
        logits = logits.detach()
        if ids is not None:
            rows = row_params.view(torch.float32).view(-1, packing.ROW_DTYPE.itemsize // 4)
            penalty = rows[:, packing.ROW_DTYPE.fields["repetition_penalty"][1] // 4].contiguous()
            logits = process_logits(logits, sample_indices=sample_indices, history_offsets=offsets, history_ids=ids,
                                    repetition_penalty=penalty, out_dtype=torch.float32)
            sample_indices = None
        return out, token_logprobs(logits, tokens, logprobs, sample_indices=sample_indices)

    # -- pre-packed device inputs (graph-capturable) ------------------------
    def sample_packed(
        self,
        logits: torch.Tensor,
        row_params: torch.Tensor,
        history_offsets: Optional[torch.Tensor],
        history_ids: Optional[torch.Tensor],
        *,
        sample_indices: Optional[torch.Tensor] = None,
        uniforms: Optional[torch.Tensor] = None,
        seed: Optional[int] = None,
        offset: Optional[int] = None,
        row_offset: int = 0,
        out: Optional[torch.Tensor] = None,
        out_dtype: torch.dtype = torch.int64,
        return_debug: bool = False,
        row_order: Optional[torch.Tensor] = None,
    ):
        """One step over pre-packed device inputs (``packing.pack`` + ``upload_packed``).

        ``row_order`` (int32 [S], a permutation) only changes the order in
        which the kernel takes rows, never the result."""
        S = row_params.numel() // packing.ROW_DTYPE.itemsize
        dev = logits.device
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        if out is None:
            out = torch.empty(S, dtype=out_dtype, device=dev)
        if seed is None:
            seed = torch.initial_seed()
        if offset is None:
            offset = self._step
            self._step += 1
        dbg = None
        if return_debug:
            V = logits.shape[1]
            dbg = {
                "penalized": torch.empty(S, V, dtype=torch.float32, device=dev),
                "filtered": torch.empty(S, V, dtype=torch.float32, device=dev),
                "probs": torch.empty(S, V, dtype=torch.float32, device=dev),
                "status": torch.zeros(1, dtype=torch.int32, device=dev),
            }
        torch.ops.nanoserve_b200.sample(
            logits, sample_indices, row_params, history_offsets, history_ids, uniforms,
            int(seed) & 0x7FFFFFFFFFFFFFFF, int(offset), int(row_offset), out,
            dbg["penalized"] if dbg else None, dbg["filtered"] if dbg else None,
            dbg["probs"] if dbg else None, dbg["status"] if dbg else None, row_order, KERNELS[self.kernel],
        )
        if return_debug:
            return out, dbg
        return out

    def _upload(self, packed: packing.Packed, device: torch.device):
        a, b, c, d, end = packing.layout(packed)
        host = self._staging.get(end)
        packing.to_bytes(packed, host.numpy())
        dev = host.to(device, non_blocking=True)
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(device))
        self._staging.event = ev
        row_params = dev[a : a + packed.row_params.nbytes]
        offsets = dev[b : b + packed.offsets.nbytes].view(torch.int64)
        ids = dev[c : c + packed.ids.nbytes].view(torch.int32) if packed.ids.size else None
        if ids is None:
            offsets = None
        order = dev[d : d + packed.order.nbytes].view(torch.int32) if packed.order is not None else None
        return row_params, offsets, ids, order


class _ListHistories:
    """Histories given as Python lists, for ``_sample_processed``."""

    def __init__(self, histories: Sequence[Sequence[int]], rows: int, vocab: int):
        if len(histories) < rows:
            raise IndexError("history_token_ids has fewer entries than sampling_params_list")
        self._histories, self._rows, self._vocab = histories, rows, vocab

    def lens(self) -> np.ndarray:
        return np.fromiter((len(self._histories[i]) for i in range(self._rows)), dtype=np.int64, count=self._rows)

    def parts(self, lens: np.ndarray) -> List[np.ndarray]:
        return [packing.flatten_histories(self._histories, lens, self._vocab)]

    def ids(self, parts: Sequence[torch.Tensor], offsets: torch.Tensor, total: int) -> torch.Tensor:
        return parts[0]


_TORCH_DTYPES = {np.dtype(np.uint8): torch.uint8, np.dtype(np.int32): torch.int32, np.dtype(np.int64): torch.int64,
                 np.dtype(np.float32): torch.float32}


def upload_parts(staging: _Staging, arrays: Sequence[np.ndarray], device: torch.device) -> List[torch.Tensor]:
    """The arrays on ``device`` (the current one), through one pinned buffer and one copy on the current stream."""
    at, end = [], 0
    for a in arrays:
        at.append(end)
        end = (end + a.nbytes + 15) & ~15
    host = staging.get(max(end, 16))
    hb = host.numpy()
    for a, o in zip(arrays, at):
        hb[o : o + a.nbytes] = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
    dev = host.to(device, non_blocking=True)
    ev = torch.cuda.Event()
    ev.record(torch.cuda.current_stream(device))
    staging.event = ev
    return [dev[o : o + a.nbytes].view(_TORCH_DTYPES[a.dtype]) for a, o in zip(arrays, at)]


def upload_packed(packed: packing.Packed, device) -> tuple:
    """Device tensors (row_params uint8, offsets int64 or None, ids int32 or
    None, row order int32 or None) for :meth:`Sampler.sample_packed`."""
    device = torch.device(device)
    rp = torch.from_numpy(packed.row_params.view(np.uint8).copy()).to(device)
    if packed.ids.size:
        off = torch.from_numpy(packed.offsets.copy()).to(device)
        ids = torch.from_numpy(packed.ids.copy()).to(device)
    else:
        off, ids = None, None
    order = torch.from_numpy(packed.order.copy()).to(device) if packed.order is not None else None
    return rp, off, ids, order


_SMS: dict = {}


def _sm_count(device) -> int:
    """SM count of a CUDA device (cached)."""
    device = torch.device(device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _SMS:
        _SMS[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _SMS[idx]
