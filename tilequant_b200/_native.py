"""ctypes binding of the C ABI in ``include/tilequant_b200.h``.

The library is ``libtilequant_b200.so`` next to this file (built by
``python -m tilequant_b200.build``).  There is no fallback: if the library is
missing, or the tensors are not on a CUDA device, the calls raise.
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libtilequant_b200.so"

TQ_OK, TQ_ERR_INVALID, TQ_ERR_UNSUPPORTED, TQ_ERR_CUDA, TQ_ERR_TIMEOUT = range(5)
TQ_DTYPE_BF16, TQ_DTYPE_F16 = 0, 1
TQ_PAGES_POOL_EMPTY, TQ_PAGES_TABLE_FULL, TQ_PAGES_ROWS_FULL, TQ_PAGES_BAD_PAGE = 1, 2, 4, 8
TQ_MAX_REQUESTS = 4096
TQ_CLEAR_REST = 1
TQ_ALGO_AUTO, TQ_ALGO_ROWS, TQ_ALGO_UMMA, TQ_ALGO_GEMV, TQ_ALGO_STREAM = 0, 1, 2, 3, 4
ABI_VERSION = 1

_P, _I64, _I, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


class AttnArgs(ctypes.Structure):
    """``tq_attn_args`` of the header, field for field."""

    _fields_ = [(name, _P) for name in ("q", "k", "v", "cos", "sin", "k_cache", "v_cache", "pos", "ws_m", "ws_l",
                                        "ws_o", "err")] + \
               [(name, _I64) for name in ("ld_q", "ld_k", "ld_v")] + \
               [(name, _I) for name in ("B", "Hq", "Hkv", "D", "L", "S")] + \
               [("scale_log2", ctypes.c_float), ("reserved", _I)]



class PlanArgs(ctypes.Structure):
    """``tq_plan_args`` of the header, field for field."""

    _fields_ = [(name, _P) for name in ("new_lens", "lengths", "lengths_out", "block_table", "free_pages", "free_count",
                                        "free_count_out", "cu_new", "slots", "positions", "kv_len", "items", "counts",
                                        "cu_work", "attn_start", "status")] + \
               [(name, _I) for name in ("requests", "table_width", "page", "pages", "max_tokens", "kv_heads", "group",
                                        "row_tile", "attn_ctas", "reserved")]


class CacheWriteArgs(ctypes.Structure):
    """``tq_cache_write_args`` of the header, field for field."""

    _fields_ = [(name, _P) for name in ("k", "v", "q", "cos", "sin", "q_out", "k_codes", "v_codes", "k_scale",
                                        "v_scale", "items", "counts", "cu_new", "status")] + \
               [(name, _I64) for name in ("ld_k", "ld_v", "ld_q", "ld_qo", "ld_cs")] + \
               [(name, _I) for name in ("rows", "requests", "pages", "page", "kv_heads", "q_heads", "head_dim",
                                        "flags")]


class PagedAttnArgs(ctypes.Structure):
    """``tq_paged_attn_args`` of the header, field for field."""

    _fields_ = [(name, _P) for name in ("q", "out", "k_codes", "v_codes", "k_scale", "v_scale", "block_table", "cu_new",
                                        "kv_len", "cu_work", "attn_start", "counts", "ws_o", "ws_ml", "arrivals", "err",
                                        "status")] + \
               [(name, _I64) for name in ("ld_q", "ld_out")] + \
               [(name, _I) for name in ("rows", "requests", "table_width", "pages", "page", "kv_heads", "q_heads",
                                        "head_dim", "row_tile", "attn_ctas")] + \
               [("scale_log2", ctypes.c_float), ("flags", _I)]


class SampleArgs(ctypes.Structure):
    """``tq_sample_args`` of the header, field for field."""

    _fields_ = [(name, _P) for name in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p", "ids", "logprobs",
                                        "keys", "next", "token", "generated", "position")] + \
               [(name, _I64) for name in ("ld", "u_ld", "u_cols", "gen_ld", "gen_cols", "prompt_tokens")] + \
               [(name, _I) for name in ("n_rows", "vocab")]


# name -> argument types, in header order
SIGNATURES = {
    "tq_abi_version": [],
    "tq_last_error": [],
    "tq_status_string": [_I],
    "tq_kernel_launches": [],
    "tq_act_scales": [_P, _I, _I64, _I64, _I64, _I64, _P, _P],
    "tq_quantize_with_scales": [_P, _I, _I64, _I64, _I64, _I64, _P, _P, _I64, _P],
    "tq_quantize_act": [_P, _I, _I64, _I64, _I64, _I64, _P, _I64, _P, _P],
    "tq_gemm_mixed": [_P, _I64, _P, _P, _P, _P, _P, _I64, _P, _I64, _P, _P, _P, _I64, _I, _P, _I64, _I, _P,
                      _I64, _I64, _I64, _I, _I, _I, _I, _P, _P],
    "tq_gemm_mixed_fused_quant": [_P, _I64, _I, _P, _P, _P, _P, _I64, _P, _P, _P, _I64, _P, _I64, _I, _P, _I64,
                                  _I64, _I64, _I, _I, _I, _P, _P],
    "tq_gemm_rows_plan": [_I64, _I, _I, _I, _I, _P, _P],
    "tq_gemm_int8_partials": [_P, _I64, _P, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I, _P],
    "tq_pack_int8_tiles": [_P, _I, _I64, _I64, _I64, _I, _P, _I64, _P, _P, _P, _P],
    "tq_gather_fp_tiles": [_P, _I, _I64, _I64, _I64, _I, _P, _I64, _P, _P],
    "tq_add_rmsnorm": [_P, _I64, _P, _I64, _P, _P, _I64, _P, _I64, _I64, _I64, _F, _I, _P],
    "tq_silu_mul_quant": [_P, _P, _I64, _I64, _I64, _P, _I64, _P, _I64, _P, _I, _P],
    "tq_attn_decode_splits": [_I, _I, _I],
    "tq_attn_decode": [ctypes.POINTER(AttnArgs), _P, _I64, _P, _I64, _P, _I, _P],
    "tq_greedy_pick": [_P, _I64, _I64, _I64, _I, _P, _P, _P, _P, _I64, _I64, _P, _I64, _P],
    "tq_plan_items": [_I64, _I, _I],
    "tq_plan_step": [ctypes.POINTER(PlanArgs), _P],
    "tq_release_requests": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
    "tq_cache_write": [ctypes.POINTER(CacheWriteArgs), _I, _P],
    "tq_read_pages": [_P, _P, _P, _P, _P, _I64, _I, _I, _I, _I, _P, _P, _I, _P],
    "tq_paged_attn_ctas": [_I],
    "tq_attn_paged": [ctypes.POINTER(PagedAttnArgs), _I, _P],
    "tq_sample": [ctypes.POINTER(SampleArgs), _I, _P],
    "tq_calib_gi_accumulate": [_P, _P, _I, _I64, _I64, _I64, _I64, _I, _I, _P, _P],
    "tq_calib_iaa_channel_accumulate": [_P, _I, _I64, _I64, _I64, _P, _P],
    "tq_calib_iaa_tile_scores": [_P, _I, _I64, _I64, _I64, _P, _I64, _P, _P, _P],
    "tq_peer_buffer_bytes": [_I, _I],
    "tq_peer_alloc": [_I, _I, _P],
    "tq_peer_free": [_P],
    "tq_peer_ipc_handle": [_P, _P],
    "tq_peer_ipc_open": [_P, _P],
    "tq_peer_ipc_close": [_P],
    "tq_peer_reset": [_P, _I, _I, _P, _P],
    "tq_gemm_mixed_peer_sum": [_P, _I64, _P, _P, _P, _P, _P, _I64, _P, _I64, _P, _P, _P, _I64, _I, _P, _I64, _I, _P,
                               _I64, _I64, _I64, _I, _I, _I, _P, _P, _I, _I, _I, _I64, _P, _P],
    "tq_gemm_mixed_peer_sum_noalloc": [_P, _I64, _P, _P, _P, _P, _P, _I64, _P, _I64, _P, _P, _P, _I64, _I, _P, _I64,
                                       _I, _P, _I64, _I64, _I64, _I, _I, _I, _I64, _I, _P, _P],
}

TQ_PEER_MAX_WORLD, TQ_PEER_MAX_SLOTS, TQ_IPC_HANDLE_BYTES = 8, 65536, 64

_lib = None
_lock = threading.Lock()


class TileQuantError(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    """Load the native library (once).  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise TileQuantError(
                    f"native library {LIB_PATH} is missing: build it with `python -m tilequant_b200.build`"
                )
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, argtypes in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = argtypes
                fn.restype = _I
            lib.tq_last_error.restype = ctypes.c_char_p
            lib.tq_status_string.restype = ctypes.c_char_p
            lib.tq_kernel_launches.restype = ctypes.c_int64
            lib.tq_peer_buffer_bytes.restype = ctypes.c_int64
            lib.tq_plan_items.restype = ctypes.c_int64
            if lib.tq_abi_version() != ABI_VERSION:
                raise TileQuantError("libtilequant_b200.so ABI version mismatch; rebuild it")
            _lib = lib
    return _lib


def check(rc: int, what: str) -> None:
    """Map a C status to the exception the reference raises for the same problem."""
    if rc == TQ_OK:
        return
    msg = load().tq_last_error().decode(errors="replace")
    if rc == TQ_ERR_INVALID:
        raise ValueError(f"{what}: {msg}")
    raise TileQuantError(f"{what}: {load().tq_status_string(rc).decode()}: {msg}")


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return TQ_DTYPE_BF16
    if dtype == torch.float16:
        return TQ_DTYPE_F16
    raise ValueError(f"unsupported 16-bit float dtype {dtype}; expected bfloat16 or float16")


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("tilequant_b200 kernels need CUDA tensors (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    return dev


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(index: int) -> int:
    """The current stream of device ``index``, without building a Stream object."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def on_device(index: int, fn, *args) -> int:
    """``fn(*args)`` with device ``index`` current."""
    if torch.cuda.current_device() == index:
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _refuse(what: str):
    def refuse(*args, **kwargs):
        raise AttributeError(f"{what} keeps its memory: copy into it")

    return refuse


class FixedTensors:
    """Base of objects whose tensor attributes stay the ones they were built with, so that
    their addresses and shapes are checked once: copy into them (or change them in place) instead
    of replacing them.

    Kernels go on using the memory of the construction: the attributes refuse ``resize_`` and
    ``set_``, and an alias keeps that memory for as long as the object lives (after ``.data =`` a
    tensor no longer shows what the kernels use)."""

    def __setattr__(self, name, value):
        if isinstance(self.__dict__.get(name), torch.Tensor):
            if value is self.__dict__[name]:  # the end of an in-place operator (x.a += 1)
                return
            raise AttributeError(f"{type(self).__name__}.{name} cannot be replaced: copy into it")
        if isinstance(value, torch.Tensor):
            self.__dict__.setdefault("_memory", []).append(value.detach())
            for method in ("resize_", "resize_as_", "set_"):
                setattr(value, method, _refuse(f"{type(self).__name__}.{name}"))
        object.__setattr__(self, name, value)

    def __reduce_ex__(self, protocol):
        raise TypeError(f"a {type(self).__name__} cannot be copied or pickled (its addresses would be the original's): "
                        "make another and copy the tensors into it")


def kernel_launches() -> int:
    """Kernels this library has launched in the process so far."""
    return int(load().tq_kernel_launches())
