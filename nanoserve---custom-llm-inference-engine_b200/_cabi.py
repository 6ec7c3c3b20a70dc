"""ctypes binding of the C ABI in ``include/nanoserve_sampler.h``.

This is the binding a Python maintainer of the reference would add to call
the library without torch's op registry: the structs mirror the header field
for field, and :func:`ns_sample` raises on a non-zero status with the
library's own message.  The library is loaded from this package directory;
a missing library raises instead of falling back to anything else.
"""
from __future__ import annotations

import ctypes
from pathlib import Path
from typing import Sequence

PKG_DIR = Path(__file__).resolve().parent
LIB_PATH = PKG_DIR / "libnanoserve_sampler.so"

NS_OK = 0
NS_ERR_INVALID_ARG = 1
NS_ERR_UNSUPPORTED = 2
NS_ERR_CUDA = 3

NS_DTYPE_F32 = 0
NS_DTYPE_BF16 = 1
NS_OUT_I64 = 0
NS_OUT_I32 = 1

NS_KERNEL_AUTO = 0
NS_KERNEL_CLUSTER = 1
NS_KERNEL_SPLIT = 2

NS_ROW_GREEDY = 0x1
NS_ROW_TOP_P = 0x2
NS_ROW_PENALTY = 0x4
NS_ROW_SEED = 0x8

NS_STATUS_BAD_SAMPLE_INDEX = 0x1
NS_STATUS_BAD_HISTORY_ID = 0x2
NS_STATUS_WAIT_TIMEOUT = 0x4
NS_STATUS_CAP_OVERFLOW = 0x8
NS_STATUS_BAD_ROW_ORDER = 0x10
NS_STATUS_BAD_POOL_RANGE = 0x20
NS_STATUS_BAD_TOKEN_ID = 0x40
NS_STATUS_BAD_ROW_RANGE = 0x80
NS_STATUS_BAD_MASK_ROW = 0x100

NS_MAX_TOP_LOGPROBS = 32

# every entry point the header declares
EXPORTED_SYMBOLS = ("ns_sample", "ns_sample_noalloc", "ns_workspace_bytes", "ns_history_gather",
                    "ns_history_append", "ns_process_logits", "ns_token_logprobs", "ns_pages_copy",
                    "ns_pages_check", "ns_pages_copy_listed",
                    "ns_paged_history_gather", "ns_last_error", "ns_abi_version", "ns_max_vocab")
NS_ABI_VERSION = 3
NS_NOALLOC_WORKSPACE_BYTES = 128


class NsRowParams(ctypes.Structure):
    _fields_ = [
        ("temperature", ctypes.c_float),
        ("top_p", ctypes.c_float),
        ("repetition_penalty", ctypes.c_float),
        ("top_k", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("seed_step", ctypes.c_uint32),
        ("seed", ctypes.c_uint64),
    ]


class NsSampleArgs(ctypes.Structure):
    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("logits_dtype", ctypes.c_int32),
        ("vocab_size", ctypes.c_int32),
        ("num_logit_rows", ctypes.c_int64),
        ("logits_row_stride", ctypes.c_int64),
        ("num_rows", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("sample_indices", ctypes.c_void_p),
        ("row_params", ctypes.c_void_p),
        ("history_offsets", ctypes.c_void_p),
        ("history_ids", ctypes.c_void_p),
        ("uniforms", ctypes.c_void_p),
        ("philox_seed", ctypes.c_uint64),
        ("philox_offset", ctypes.c_uint64),
        ("row_offset", ctypes.c_int64),
        ("out_tokens", ctypes.c_void_p),
        ("out_penalized", ctypes.c_void_p),
        ("out_filtered", ctypes.c_void_p),
        ("out_probs", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("row_order", ctypes.c_void_p),
        ("kernel", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
    ]


class NsProcessArgs(ctypes.Structure):
    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("logits_dtype", ctypes.c_int32),
        ("vocab_size", ctypes.c_int32),
        ("num_logit_rows", ctypes.c_int64),
        ("logits_row_stride", ctypes.c_int64),
        ("num_rows", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("sample_indices", ctypes.c_void_p),
        ("history_offsets", ctypes.c_void_p),
        ("history_ids", ctypes.c_void_p),
        ("num_history_ids", ctypes.c_int64),
        ("prompt_lens", ctypes.c_void_p),
        ("repetition_penalty", ctypes.c_void_p),
        ("presence_penalty", ctypes.c_void_p),
        ("frequency_penalty", ctypes.c_void_p),
        ("bias_offsets", ctypes.c_void_p),
        ("bias_ids", ctypes.c_void_p),
        ("bias_values", ctypes.c_void_p),
        ("num_biases", ctypes.c_int64),
        ("allowed", ctypes.c_void_p),
        ("mask_stride", ctypes.c_int64),
        ("num_masks", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("allowed_rows", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("out_row_stride", ctypes.c_int64),
        ("status", ctypes.c_void_p),
    ]


class NsLogprobArgs(ctypes.Structure):
    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("logits_dtype", ctypes.c_int32),
        ("vocab_size", ctypes.c_int32),
        ("num_logit_rows", ctypes.c_int64),
        ("logits_row_stride", ctypes.c_int64),
        ("num_rows", ctypes.c_int32),
        ("ids_dtype", ctypes.c_int32),
        ("sample_indices", ctypes.c_void_p),
        ("token_ids", ctypes.c_void_p),
        ("top_n", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("out_logprobs", ctypes.c_void_p),
        ("out_ranks", ctypes.c_void_p),
        ("out_top_ids", ctypes.c_void_p),
        ("out_top_logprobs", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class NsPagePool(ctypes.Structure):
    _fields_ = [
        ("base", ctypes.c_void_p),
        ("page_stride", ctypes.c_int64),
        ("page_bytes", ctypes.c_int64),
    ]


assert ctypes.sizeof(NsRowParams) == 32


class NativeLibraryMissing(RuntimeError):
    """The CUDA library was not built; there is no fallback implementation."""


_lib = None


def load_library() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise NativeLibraryMissing(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(there is no CPU fallback for the sampling op)"
            )
        lib = ctypes.CDLL(str(LIB_PATH))
        lib.ns_sample.argtypes = [ctypes.POINTER(NsSampleArgs), ctypes.c_void_p]
        lib.ns_sample.restype = ctypes.c_int
        lib.ns_sample_noalloc.argtypes = [ctypes.POINTER(NsSampleArgs), ctypes.c_void_p]
        lib.ns_sample_noalloc.restype = ctypes.c_int
        lib.ns_history_gather.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p,
                                          ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        lib.ns_history_gather.restype = ctypes.c_int
        lib.ns_history_append.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p,
                                          ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]
        lib.ns_history_append.restype = ctypes.c_int
        lib.ns_process_logits.argtypes = [ctypes.POINTER(NsProcessArgs), ctypes.c_void_p]
        lib.ns_process_logits.restype = ctypes.c_int
        lib.ns_token_logprobs.argtypes = [ctypes.POINTER(NsLogprobArgs), ctypes.c_void_p]
        lib.ns_token_logprobs.restype = ctypes.c_int
        lib.ns_pages_copy.argtypes = [ctypes.POINTER(NsPagePool), ctypes.c_int32, ctypes.c_int64,
                                      ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64),
                                      ctypes.c_int64, ctypes.c_void_p]
        lib.ns_pages_copy.restype = ctypes.c_int
        lib.ns_pages_check.argtypes = [ctypes.c_int64, ctypes.POINTER(ctypes.c_int64),
                                       ctypes.POINTER(ctypes.c_int64), ctypes.c_int64]
        lib.ns_pages_check.restype = ctypes.c_int
        lib.ns_pages_copy_listed.argtypes = [ctypes.POINTER(NsPagePool), ctypes.c_int32, ctypes.c_int64,
                                             ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                             ctypes.c_void_p]
        lib.ns_pages_copy_listed.restype = ctypes.c_int
        lib.ns_paged_history_gather.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p,
                                                ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32,
                                                ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]
        lib.ns_paged_history_gather.restype = ctypes.c_int
        lib.ns_last_error.argtypes = []
        lib.ns_last_error.restype = ctypes.c_char_p
        lib.ns_abi_version.argtypes = []
        lib.ns_abi_version.restype = ctypes.c_int
        lib.ns_max_vocab.argtypes = [ctypes.c_int32]
        lib.ns_max_vocab.restype = ctypes.c_int32
        lib.ns_workspace_bytes.argtypes = [ctypes.c_int32]
        lib.ns_workspace_bytes.restype = ctypes.c_int64
        _lib = lib
    return _lib


class NsError(RuntimeError):
    def __init__(self, code: int, message: str, entry: str = "ns_sample"):
        super().__init__(f"{entry} failed ({code}): {message}")
        self.code = code


def _call(entry: str, *args) -> None:
    lib = load_library()
    rc = getattr(lib, entry)(*args)
    if rc != NS_OK:
        raise NsError(rc, lib.ns_last_error().decode(errors="replace"), entry)


def ns_sample(args: NsSampleArgs, stream: int = 0) -> None:
    lib = load_library()
    rc = lib.ns_sample(ctypes.byref(args), ctypes.c_void_p(stream))
    if rc != NS_OK:
        raise NsError(rc, lib.ns_last_error().decode(errors="replace"))


def ns_sample_noalloc(args: NsSampleArgs, stream: int = 0) -> None:
    """The entry point for callers that cannot allocate device memory: it
    ignores ``args.workspace`` and runs on the library's static workspace."""
    lib = load_library()
    rc = lib.ns_sample_noalloc(ctypes.byref(args), ctypes.c_void_p(stream))
    if rc != NS_OK:
        raise NsError(rc, lib.ns_last_error().decode(errors="replace"))


def ns_workspace_bytes(num_rows: int) -> int:
    """Bytes of ``NsSampleArgs.workspace`` for calls of up to ``num_rows`` rows."""
    return int(load_library().ns_workspace_bytes(int(num_rows)))


def ns_history_gather(pool: int, pool_size: int, row_src: int, offsets: int, num_rows: int, out_ids: int,
                      status: int = 0, stream: int = 0) -> None:
    """Build one step's CSR history ids from a device pool (device pointers as ints)."""
    lib = load_library()
    rc = lib.ns_history_gather(pool or None, pool_size, row_src or None, offsets or None, num_rows,
                               out_ids or None, status or None, ctypes.c_void_p(stream))
    if rc != NS_OK:
        raise NsError(rc, lib.ns_last_error().decode(errors="replace"))


def ns_history_append(pool: int, pool_size: int, row_dst: int, tokens: int, tokens_dtype: int, num_rows: int,
                      status: int = 0, stream: int = 0) -> None:
    """Append one sampled id per row to the device pool (device pointers as ints)."""
    lib = load_library()
    rc = lib.ns_history_append(pool or None, pool_size, row_dst or None, tokens or None, tokens_dtype, num_rows,
                               status or None, ctypes.c_void_p(stream))
    if rc != NS_OK:
        raise NsError(rc, lib.ns_last_error().decode(errors="replace"))


def ns_process_logits(args: NsProcessArgs, stream: int = 0) -> None:
    """Penalties, biases and masks on one step's logits."""
    _call("ns_process_logits", ctypes.byref(args), ctypes.c_void_p(stream))


def ns_token_logprobs(args: NsLogprobArgs, stream: int = 0) -> None:
    """Log-probabilities and ranks of one token per row, and each row's largest."""
    _call("ns_token_logprobs", ctypes.byref(args), ctypes.c_void_p(stream))


def ns_pages_copy(pools: Sequence, num_pages: int, src: Sequence[int], dst: Sequence[int], stream: int = 0) -> None:
    """Copy pages src[j] to dst[j] of every pool (``NsPagePool`` or (base, stride, bytes))."""
    if len(src) != len(dst):
        raise ValueError("src and dst must have the same number of pages")
    p = (NsPagePool * max(1, len(pools)))(*[x if isinstance(x, NsPagePool) else NsPagePool(*x) for x in pools])
    n = len(src)
    ids = ctypes.c_int64 * max(1, n)
    _call("ns_pages_copy", p, len(pools), num_pages, ids(*src), ids(*dst), n, ctypes.c_void_p(stream))


def ns_pages_check(num_pages: int, src: Sequence[int], dst: Sequence[int]) -> None:
    """The check of the page numbers that ``ns_pages_copy`` makes."""
    if len(src) != len(dst):
        raise ValueError("src and dst must have the same number of pages")
    ids = ctypes.c_int64 * max(1, len(src))
    _call("ns_pages_check", num_pages, ids(*src), ids(*dst), len(src))


def ns_pages_copy_listed(pools: Sequence, num_pages: int, src: int, dst: int, count: int, status: int = 0,
                         stream: int = 0) -> None:
    """``ns_pages_copy`` with the page numbers in device memory (int32, device pointers as ints)."""
    p = (NsPagePool * max(1, len(pools)))(*[x if isinstance(x, NsPagePool) else NsPagePool(*x) for x in pools])
    _call("ns_pages_copy_listed", p, len(pools), num_pages, src or None, dst or None, count, status or None,
          ctypes.c_void_p(stream))


def ns_paged_history_gather(pool: int, num_pages: int, page_size: int, pages: int, num_table_pages: int,
                            page_offsets: int, offsets: int, num_rows: int, out_ids: int, num_ids: int,
                            status: int = 0, stream: int = 0) -> None:
    """Build one step's CSR history ids out of pages (device pointers as ints)."""
    _call("ns_paged_history_gather", pool or None, num_pages, page_size, pages or None, num_table_pages,
          page_offsets or None, offsets or None, num_rows, out_ids or None, num_ids, status or None,
          ctypes.c_void_p(stream))
