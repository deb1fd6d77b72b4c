"""ctypes binding of the paged cache's C ABI (include/chill_cache.h), library ``_lib/libchill_cache_b200.so``."""
from __future__ import annotations

import ctypes as C
import os
import threading

from . import _cabi
from ._cabi import _S3, _S4, ChillLibraryError, MaskDesc

DEFAULT_LIB = os.path.join(_cabi.LIB_DIR, "libchill_cache_b200.so")
ABI_VERSION = 1
#: answers of chill_cached_kernel
CACHED_CUDA_CORES, CACHED_ROWS, CACHED_TILES = range(3)

EXPORTS = (
    "chill_pages_reserve", "chill_pages_reserve_stored", "chill_pages_trim", "chill_cache_append", "chill_cache_commit",
    "chill_cached_workspace_bytes", "chill_cached_fwd", "chill_cached_kernel", "chill_cache_read_device_status", "chill_cache_launch_count",
    "chill_cache_last_cuda_error", "chill_cache_abi_version",
)


class PagesArgs(C.Structure):
    _fields_ = [("B", C.c_int32), ("N", C.c_int32), ("page_size", C.c_int32), ("num_pages", C.c_int32), ("table_width", C.c_int32),
                ("reserved", C.c_int32), ("table", C.c_void_p), ("table_stride", C.c_int64), ("held", C.c_void_p),
                ("free_pages", C.c_void_p), ("n_free", C.c_void_p), ("missing", C.c_void_p), ("lens", C.c_void_p),
                ("new_lens", C.c_void_p), ("parents", C.c_void_p), ("slots", C.c_void_p), ("positions", C.c_void_p),
                ("ancestors", C.c_void_p)]


class CacheRowsArgs(C.Structure):
    _fields_ = [("B", C.c_int32), ("H_kv", C.c_int32), ("N", C.c_int32), ("D", C.c_int32), ("dtype", C.c_int32),
                ("page_size", C.c_int32), ("num_pages", C.c_int32), ("table_width", C.c_int32), ("A", C.c_int32),
                ("reserved", C.c_int32), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("k_cache_strides", _S4),
                ("v_cache_strides", _S4), ("k", C.c_void_p), ("v", C.c_void_p), ("k_strides", _S4), ("v_strides", _S4),
                ("slots", C.c_void_p), ("table", C.c_void_p), ("table_stride", C.c_int64), ("lens", C.c_void_p),
                ("new_lens", C.c_void_p), ("path", C.c_void_p), ("accepted", C.c_void_p), ("out_lens", C.c_void_p)]


class CachedArgs(C.Structure):
    _fields_ = [("mask", MaskDesc), ("B", C.c_int32), ("H", C.c_int32), ("H_kv", C.c_int32), ("N", C.c_int32), ("D", C.c_int32),
                ("dtype", C.c_int32), ("page_size", C.c_int32), ("num_pages", C.c_int32), ("table_width", C.c_int32),
                ("sm_scale", C.c_float), ("flags", C.c_uint32), ("reserved", C.c_int32), ("q", C.c_void_p),
                ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("o", C.c_void_p), ("lse", C.c_void_p), ("q_strides", _S4),
                ("k_cache_strides", _S4), ("v_cache_strides", _S4), ("o_strides", _S4), ("lse_strides", _S3),
                ("table", C.c_void_p), ("table_stride", C.c_int64), ("lens", C.c_void_p), ("new_lens", C.c_void_p),
                ("positions", C.c_void_p), ("ancestors", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


_libs: dict[str, C.CDLL] = {}
_lock = threading.Lock()


def load_library(path: str | None = None) -> C.CDLL:
    """dlopen the library (cached per path) and declare its prototypes."""
    path = os.path.abspath(path or DEFAULT_LIB)
    with _lock:
        lib = _libs.get(path)
        if lib is not None:
            return lib
        if not os.path.exists(path):
            raise ChillLibraryError(f"{path} not found: build the CUDA libraries first (python chill-attention_b200/build.py)")
        lib = C.CDLL(path)
        for name, args in (("chill_pages_reserve", PagesArgs), ("chill_pages_trim", PagesArgs), ("chill_cache_append", CacheRowsArgs),
                           ("chill_cache_commit", CacheRowsArgs), ("chill_cached_fwd", CachedArgs)):
            getattr(lib, name).argtypes = [C.POINTER(args), C.c_void_p]
            getattr(lib, name).restype = C.c_int
        lib.chill_pages_reserve_stored.argtypes = [C.POINTER(PagesArgs), C.c_void_p, C.c_void_p]
        lib.chill_pages_reserve_stored.restype = C.c_int
        lib.chill_cached_workspace_bytes.argtypes = [C.POINTER(CachedArgs)]
        lib.chill_cached_workspace_bytes.restype = C.c_size_t
        lib.chill_cached_kernel.argtypes = [C.POINTER(CachedArgs)]
        lib.chill_cache_launch_count.restype = C.c_ulonglong
        lib.chill_cache_last_cuda_error.restype = C.c_char_p
        for name in ("chill_cached_kernel", "chill_cache_read_device_status", "chill_cache_abi_version"):
            getattr(lib, name).restype = C.c_int
        if lib.chill_cache_abi_version() != ABI_VERSION:
            raise ChillLibraryError(f"{path}: ABI version {lib.chill_cache_abi_version()} != {ABI_VERSION}")
        _libs[path] = lib
        return lib
