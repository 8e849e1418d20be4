"""ctypes binding of libdsa_kv.so (C ABI: include/dsa_kv.h), and the argument
checks that its Python operators (qk_rope.py, kv_cache.py, dsa_attention.py)
share.

Loading fails loudly: there is no CPU or eager-PyTorch fallback behind this
module. If the library is missing, build it with
``python -m flagos_kernelgen_72h_shanghai_2026_b200._build``.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

from ._build import KV_LIB_PATH

try:  # C++ launch path (csrc/farq_fast.cpp); without it every call takes the ctypes path
    from . import _farq_fast as _extension
except ImportError:
    _extension = None

# enum dsa_kv_dtype
DTYPE_BF16, DTYPE_FP16, DTYPE_FP32, DTYPE_INT8, DTYPE_E4M3, DTYPE_INT32, DTYPE_INT64 = range(7)

# enum dsa_kv_status
OK = 0
ERR_NULL_POINTER = 1
ERR_BAD_SHAPE = 2
ERR_BAD_HEAD_DIM = 3
ERR_BAD_DTYPE = 4
ERR_ALIGNMENT = 5
ERR_UNSUPPORTED = 6
ERR_CUDA = 7
ERR_BAD_ARGS_SIZE = 8
ERR_DEVICE_TIMEOUT = 9

ABI_VERSION = 2


def launch_path(extension):
    """The extension module, or None where it lacks this version's entry points: one built before they were
    added, or next to a library of another version."""
    if getattr(extension, "kv_abi_version", None) != ABI_VERSION:
        return None
    return extension if all(hasattr(extension, n) for n in ("kv_rope", "kv_copy", "kv_attn")) else None


_fast = launch_path(_extension)

HALF_DTYPES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_FP16}
GAMMA_DTYPES = {**HALF_DTYPES, torch.float32: DTYPE_FP32}
CODE_DTYPES = {torch.int8: DTYPE_INT8, torch.float8_e4m3fn: DTYPE_E4M3}
INDEX_DTYPES = {torch.int32: DTYPE_INT32, torch.int64: DTYPE_INT64}


class Dense(ctypes.Structure):
    """Mirror of dsa_kv_dense_t."""

    _fields_ = [("ptr", ctypes.c_void_p), ("stride_b", ctypes.c_int64),
                ("stride_q", ctypes.c_int64), ("stride_h", ctypes.c_int64)]


class Cache(ctypes.Structure):
    """Mirror of dsa_kv_cache_t."""

    _fields_ = [
        ("code_dtype", ctypes.c_int32), ("reserved0", ctypes.c_int32),
        ("P", ctypes.c_int64), ("H", ctypes.c_int64), ("block_size", ctypes.c_int64),
        ("D", ctypes.c_int64),
        ("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
        ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
        ("k_scale_stride", ctypes.c_int64 * 3), ("v_scale_stride", ctypes.c_int64 * 3),
    ]


class RopeArgs(ctypes.Structure):
    """Mirror of dsa_kv_rope_args_t."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("gamma_dtype", ctypes.c_int32), ("pos_dtype", ctypes.c_int32),
        ("interleaved", ctypes.c_int32), ("eps", ctypes.c_float),
        ("B", ctypes.c_int64), ("Q", ctypes.c_int64), ("Hq", ctypes.c_int64),
        ("Hk", ctypes.c_int64), ("D", ctypes.c_int64), ("rot", ctypes.c_int64),
        ("max_pos", ctypes.c_int64),
        ("q", Dense), ("k", Dense), ("q_out", Dense), ("k_out", Dense),
        ("q_gamma", ctypes.c_void_p), ("k_gamma", ctypes.c_void_p),
        ("cos_sin", ctypes.c_void_p), ("positions", ctypes.c_void_p),
    ]


class CopyArgs(ctypes.Structure):
    """Mirror of dsa_kv_copy_args_t."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("page_dtype", ctypes.c_int32), ("pos_dtype", ctypes.c_int32),
        ("B", ctypes.c_int64), ("Q", ctypes.c_int64), ("NB", ctypes.c_int64),
        ("k", Dense), ("v", Dense), ("cache", Cache),
        ("page_table", ctypes.c_void_p), ("pos", ctypes.c_void_p),
    ]


class AttnArgs(ctypes.Structure):
    """Mirror of dsa_kv_attn_args_t."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("block_dtype", ctypes.c_int32), ("page_dtype", ctypes.c_int32),
        ("pos_dtype", ctypes.c_int32), ("softmax_scale", ctypes.c_float),
        ("B", ctypes.c_int64), ("Q", ctypes.c_int64), ("G", ctypes.c_int64),
        ("K", ctypes.c_int64),
        ("q", Dense), ("out", Dense), ("cache", Cache),
        ("blocks", ctypes.c_void_p), ("pages", ctypes.c_void_p),
        ("blocks_stride", ctypes.c_int64 * 3), ("pages_stride", ctypes.c_int64 * 3),
        ("q_pos", ctypes.c_void_p), ("kv_lens", ctypes.c_void_p), ("lse", ctypes.c_void_p),
    ]


_lock = threading.Lock()
_lib = None
_LAUNCHES = {"dsa_kv_rope_launch": RopeArgs, "dsa_kv_write_launch": CopyArgs,
             "dsa_kv_read_launch": CopyArgs, "dsa_kv_attn_launch": AttnArgs}


def load(path: Path | str | None = None) -> ctypes.CDLL:
    """Load libdsa_kv.so once and declare its prototypes. Raises if it is absent."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    with _lock:
        if _lib is not None and path is None:
            return _lib
        p = Path(path) if path is not None else KV_LIB_PATH
        if not p.exists():
            raise RuntimeError(
                f"libdsa_kv.so not found at {p}; the CUDA path has no fallback. "
                "Build it with: python -m flagos_kernelgen_72h_shanghai_2026_b200._build"
            )
        lib = ctypes.CDLL(str(p))
        lib.dsa_kv_abi_version.argtypes = []
        lib.dsa_kv_abi_version.restype = ctypes.c_int
        v = lib.dsa_kv_abi_version()
        if v != ABI_VERSION:
            raise RuntimeError(f"libdsa_kv.so ABI version {v} != expected {ABI_VERSION}; rebuild it")
        for name, args in _LAUNCHES.items():
            fn = getattr(lib, name)
            fn.argtypes = [ctypes.POINTER(args), ctypes.c_void_p]
            fn.restype = ctypes.c_int
        lib.dsa_kv_attn_launch_status.argtypes = [ctypes.POINTER(AttnArgs), ctypes.c_void_p,
                                                  ctypes.c_int32, ctypes.c_void_p]
        lib.dsa_kv_attn_launch_status.restype = ctypes.c_int
        lib.dsa_kv_strerror.argtypes = [ctypes.c_int]
        lib.dsa_kv_strerror.restype = ctypes.c_char_p
        if path is None:
            _lib = lib
        return lib


def strerror(status: int) -> str:
    return load().dsa_kv_strerror(status).decode()


def raise_status(op: str, status: int):
    msg = f"{op}: {strerror(status)}"
    if status == ERR_BAD_DTYPE:
        raise TypeError(msg)
    if status in (ERR_CUDA, ERR_BAD_ARGS_SIZE):
        raise RuntimeError(msg)
    raise ValueError(msg)


def launch(op: str, entry: str, args, device: torch.device, *more) -> None:
    """Call a C entry point on the device's current stream; raise its error."""
    fn = getattr(load(), entry)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        st = fn(ctypes.byref(args), *more, ctypes.c_void_p(stream))
    if st != OK:
        raise_status(op, st)


# ------------------------------------------------------------ argument checks
def check_tensor(name: str, t, device: torch.device | None) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise TypeError(f"{name} is on {t.device}; CUDA tensors only")
    if device is not None and t.device != device:
        raise TypeError(f"{name} is on {t.device}, expected {device}")
    return t.device


def check_shape(name: str, t: torch.Tensor, shape) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")


def dtype_code(name: str, t: torch.Tensor, codes: dict) -> int:
    code = codes.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be one of {', '.join(str(d) for d in codes)}, got {t.dtype}")
    return code


def check_contiguous(name: str, t: torch.Tensor) -> None:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def dense(name: str, t: torch.Tensor, shape, dtype: torch.dtype, device: torch.device) -> Dense:
    """A [B, Q, H, D] tensor whose last dimension is contiguous."""
    check_tensor(name, t, device)
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    check_shape(name, t, shape)
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return Dense(t.data_ptr() or None, *t.stride()[:3])


def cache(k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor,
          v_scale: torch.Tensor, device: torch.device) -> Cache:
    """Codes [P, H, block_size, D] and scales [P, H, block_size] of keys and values."""
    for name, t in (("k_cache", k_cache), ("k_scale", k_scale), ("v_cache", v_cache),
                    ("v_scale", v_scale)):
        check_tensor(name, t, device)
    code = dtype_code("k_cache", k_cache, CODE_DTYPES)
    if v_cache.dtype != k_cache.dtype:
        raise TypeError(f"v_cache must have k_cache's dtype {k_cache.dtype}, got {v_cache.dtype}")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be [P, H, block_size, D], got {list(k_cache.shape)}")
    check_shape("v_cache", v_cache, k_cache.shape)
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        check_shape(name, t, k_cache.shape[:3])
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous along its last dimension")
    three = ctypes.c_int64 * 3
    return Cache(code, 0, *k_cache.shape, k_cache.data_ptr() or None, v_cache.data_ptr() or None,
                 k_scale.data_ptr() or None, v_scale.data_ptr() or None,
                 three(*k_cache.stride()[:3]), three(*v_cache.stride()[:3]),
                 three(*k_scale.stride()), three(*v_scale.stride()))
