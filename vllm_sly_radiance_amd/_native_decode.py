"""Loading of libdecode_ops.so (C ABI: include/decode_ops.h): ops(), its binding to torch tensors, and
lib(), the C functions through ctypes. Loaded as _native loads the linear path's library: after torch, with
no fallback. A missing or stale library raises, and so does every nonzero status (RuntimeError carrying
dec_last_error())."""
from __future__ import annotations

import ctypes
import importlib
import os
import threading

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libdecode_ops.so")
ABI_VERSION = 1
SILU, BF16, LOGPROBS = 1, 2, 4

_c = ctypes
_vp, _int, _long, _sz, _f = _c.c_void_p, _c.c_int, _c.c_long, _c.c_size_t, _c.c_float
_psz = _c.POINTER(_c.c_size_t)

# name -> (restype, argtypes); the exported surface, checked against the header by the tests
SIGNATURES = {
    "dec_abi_version": (_int, []),
    "dec_last_error": (_c.c_char_p, []),
    "dec_causal_conv": (_int, [_vp, _long, _vp, _vp, _vp, _long, _long, _vp, _vp, _vp, _long, _int, _vp,
                               _int, _int, _int, _int, _int, _int, _vp]),
    "dec_gated_delta": (_int, [_vp, _long, _long, _vp, _long, _long, _vp, _long, _long, _vp, _long, _vp,
                               _long, _vp, _vp, _vp, _long, _long, _vp, _vp, _vp, _long, _int, _vp, _vp,
                               _sz, _int, _int, _int, _int, _int, _int, _int, _f, _f, _vp]),
    "dec_gated_delta_workspace": (_int, [_int] * 8 + [_psz]),
    "dec_sample": (_int, [_vp, _long, _vp, _vp, _f, _vp, _int, _vp, _f, _vp, _f, _vp, _vp, _vp, _sz,
                          _int, _int, _int, _vp]),
    "dec_sample_workspace": (_int, [_int, _int, _int, _int, _psz]),
}

_lock = threading.Lock()
_lib = _ops = None


def load_cdll(path: str = LIB_PATH) -> ctypes.CDLL:
    """dlopen the library and declare every signature (no GPU needed)."""
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is not built: run __graft_entry__.build() "
                           "(hipcc --offload-arch=gfx950) first")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    if lib.dec_abi_version() != ABI_VERSION:
        raise RuntimeError(f"{path}: ABI {lib.dec_abi_version()} != expected {ABI_VERSION}")
    return lib


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                import torch  # noqa: F401  (bind to torch's HIP runtime before dlopen)
                _lib = load_cdll()
    return _lib


def ops():
    """The ops on torch tensors (csrc/decode_torch.cpp)."""
    global _ops
    if _ops is None:
        lib()                       # raises where it is not built, or not this ABI
        try:
            _ops = importlib.import_module("._decode_torch", __package__)
        except ImportError as e:
            raise RuntimeError("_decode_torch.so is not built for this torch: run "
                               f"__graft_entry__.build() first ({e})") from e
    return _ops


def check(rc: int) -> None:
    if rc != 0:
        raise RuntimeError("[radiance.decode] " + lib().dec_last_error().decode(errors="replace"))


def gated_delta_workspace(total, batch, max_q, write_cols, k_heads, v_heads, dk, dv) -> int:
    n = _sz()
    check(lib().dec_gated_delta_workspace(total, batch, max_q, write_cols, k_heads, v_heads, dk, dv,
                                          _c.byref(n)))
    return n.value


def sample_workspace(rows, vocabulary, top_k, flags) -> int:
    n = _sz()
    check(lib().dec_sample_workspace(rows, vocabulary, top_k, flags, _c.byref(n)))
    return n.value
