"""ctypes binding of include/chill_decode.h, library ``_lib/libchill_decode_b200.so``: rotary positions, beam selection, shared pages."""
from __future__ import annotations

import ctypes as C
import os
import threading

from . import _cabi
from ._cabi import _S3, _S4, ChillLibraryError

DEFAULT_LIB = os.path.join(_cabi.LIB_DIR, "libchill_decode_b200.so")
ABI_VERSION = 1
#: most beams of a group, and most candidates that a selection keeps
SELECT_MAX = 64
#: most requests of a fork
FORK_MAX = 8192

EXPORTS = (
    "chill_rotate", "chill_rotate_append", "chill_beam_select", "chill_select_workspace_bytes", "chill_pages_fork", "chill_pages_trim_shared",
    "chill_pages_compact", "chill_share_workspace_bytes", "chill_cache_copy", "chill_decode_launch_count", "chill_decode_last_cuda_error", "chill_decode_abi_version",
)

_S5 = C.c_int64 * 5


class RotateArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("B", "H", "H_kv", "L", "D", "dtype", "pairs", "n_axes", "interleaved", "inverse")] + \
               [("inv_freq", C.c_void_p), ("axes", C.c_void_p), ("positions", C.c_void_p), ("position_strides", _S3), ("q", C.c_void_p),
                ("k", C.c_void_p), ("q_strides", _S4), ("k_strides", _S4), ("q_out", C.c_void_p), ("k_out", C.c_void_p),
                ("q_out_strides", _S4), ("k_out_strides", _S4), ("v", C.c_void_p), ("v_strides", _S4), ("k_cache", C.c_void_p),
                ("v_cache", C.c_void_p), ("k_cache_strides", _S4), ("v_cache_strides", _S4), ("slots", C.c_void_p),
                ("num_pages", C.c_int32), ("page_size", C.c_int32)]


class SelectArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("G", "K", "M", "dtype")] + \
               [("V", C.c_int64), ("logits", C.c_void_p), ("row_stride", C.c_int64), ("scores", C.c_void_p), ("finished", C.c_void_p),
                ("end_token", C.c_int64), ("out_scores", C.c_void_p), ("out_rows", C.c_void_p), ("out_tokens", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class ShareArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("B", "page_size", "num_pages", "table_width")] + \
               [("table", C.c_void_p), ("table_stride", C.c_int64)] + \
               [(n, C.c_void_p) for n in ("held", "free_pages", "n_free", "shared", "lens", "missing", "parents", "out_lens", "source", "target",
                                          "rows", "count", "workspace")] + [("workspace_bytes", C.c_size_t)]


class CopyArgs(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("layers", "num_pages", "H_kv", "page_size", "D", "dtype")] + \
               [("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("k_cache_strides", _S5), ("v_cache_strides", _S5)] + \
               [(n, C.c_void_p) for n in ("source", "target", "rows", "count")] + [("orders", C.c_int32), ("reserved", C.c_int32)]


_lib: C.CDLL | None = None
_lock = threading.Lock()


def load_library(path: str | None = None) -> C.CDLL:
    """dlopen the library (kept, where it is the default one) and declare its prototypes."""
    global _lib
    with _lock:
        if _lib is not None and path in (None, DEFAULT_LIB):
            return _lib
        found = os.path.abspath(path or DEFAULT_LIB)
        if not os.path.exists(found):
            raise ChillLibraryError(f"{found} not found: build the CUDA libraries first (python chill-attention_b200/build.py)")
        lib = C.CDLL(found)
        for name, args in (("chill_rotate", RotateArgs), ("chill_rotate_append", RotateArgs), ("chill_beam_select", SelectArgs),
                           ("chill_pages_fork", ShareArgs), ("chill_pages_trim_shared", ShareArgs), ("chill_pages_compact", ShareArgs),
                           ("chill_cache_copy", CopyArgs)):
            getattr(lib, name).argtypes = [C.POINTER(args), C.c_void_p]
            getattr(lib, name).restype = C.c_int
        for name, args in (("chill_share_workspace_bytes", ShareArgs), ("chill_select_workspace_bytes", SelectArgs)):
            getattr(lib, name).argtypes = [C.POINTER(args)]
            getattr(lib, name).restype = C.c_size_t
        lib.chill_decode_launch_count.restype = C.c_ulonglong
        lib.chill_decode_last_cuda_error.restype = C.c_char_p
        lib.chill_decode_abi_version.restype = C.c_int
        if lib.chill_decode_abi_version() != ABI_VERSION:
            raise ChillLibraryError(f"{found}: ABI version {lib.chill_decode_abi_version()} != {ABI_VERSION}")
        if path in (None, DEFAULT_LIB):
            _lib = lib
        return lib
