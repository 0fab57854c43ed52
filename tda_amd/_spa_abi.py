"""ctypes binding of the paged cache (include/spa.h) in libtda_hip.so."""
from __future__ import annotations

import ctypes
import threading

from . import _abi, _sda_abi
from ._abi import TdaTensor

ABI_VERSION = 1

ERR_PAGES = -30
ERR_ROWS = -31

_i32, _i64, _p = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class SpaCache(ctypes.Structure):
    _fields_ = [(n, _i64) for n in ("pages", "kv_heads", "page_size", "head_dim", "v_head_dim")] + [(n, _p) for n in ("k1", "k2", "v")]


class SpaRows(ctypes.Structure):
    _fields_ = [("sequences", _i64), ("rows", _i64), ("table", _p), ("table_stride", _i64), ("table_len", _i64),
                ("lengths", _p), ("starts", _p), ("counts", _p)]


_HEAD = [("abi_version", _i32), ("dtype", _i32), ("cache", SpaCache), ("at", SpaRows)]


class SpaAppendArgs(ctypes.Structure):
    _fields_ = _HEAD + [("k1", TdaTensor), ("k2", TdaTensor), ("v", TdaTensor), ("heads", _i64), ("q1", TdaTensor),
                        ("q2", TdaTensor), ("q1_out", TdaTensor), ("q2_out", TdaTensor), ("rot", _i64), ("axes", _i32),
                        ("sections", _i32 * _sda_abi.MAX_AXES), ("interleaved", _i32), ("position_dtype", _i32),
                        ("positions", _p), ("position_stride", _i64 * 3), ("inv_freq", _p)]


class SpaAttendArgs(ctypes.Structure):
    _fields_ = _HEAD + [("heads", _i64), ("most", _i64), ("scale", ctypes.c_float), ("lambda_dtype", _i32), ("q1", TdaTensor),
                        ("q2", TdaTensor), ("out", TdaTensor), ("lambda_param", _p), ("lambda_stride", _i64 * 3),
                        ("workspace", _p), ("workspace_bytes", ctypes.c_size_t)]


# Every function include/spa.h declares: name -> (restype, argtypes)
SIGNATURES = {
    "spa_abi_version": (_i32, []),
    "spa_error_string": (ctypes.c_char_p, [_i32]),
    "spa_attend_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(SpaAttendArgs)]),
    "spa_validate_append": (_i32, [ctypes.POINTER(SpaAppendArgs)]),
    "spa_validate_attend": (_i32, [ctypes.POINTER(SpaAttendArgs)]),
    "spa_append": (_i32, [ctypes.POINTER(SpaAppendArgs), _p]),
    "spa_attend": (_i32, [ctypes.POINTER(SpaAttendArgs), _p]),
}

_lock = threading.Lock()
_lib = None


def load():
    """The library with these functions bound (RuntimeError when it is missing or older)."""
    global _lib
    if _lib is not None:
        return _lib
    lib = _sda_abi.load()
    with _lock:
        for name, (res, args) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError:
                raise RuntimeError(f"tda_amd: {_abi.lib_path()} has no {name}; build it again with "
                                   "`python -m tda_amd.build`") from None
            fn.restype, fn.argtypes = res, args
        v = lib.spa_abi_version()
        if v != ABI_VERSION:
            raise RuntimeError(f"tda_amd: {_abi.lib_path()} has paged cache ABI version {v}, expected {ABI_VERSION}")
        _lib = lib
    return _lib


def check(code: int, what: str) -> None:
    """Argument errors -> ValueError, launch failures -> TdaError (a RuntimeError)."""
    if code == _abi.OK:
        return
    lib = load()
    msg = f"{what}: {lib.spa_error_string(code).decode()} (code {code})"
    if code == _abi.ERR_HIP:
        raise _abi.TdaError(code, f"{msg}; hipError_t {lib.tda_last_hip_error()}")
    raise ValueError(msg)
