"""ctypes binding of the layer norm (include/sln.h) in libtda_hip.so."""
from __future__ import annotations

import ctypes
import threading

from . import _abi, _sda_abi
from ._abi import TdaTensor

ABI_VERSION = 1
MAX_WIDTH = 16384

ERR_WIDTH = -40
ERR_EPS = -41

_i32, _i64, _p = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p

_HEAD = [("abi_version", _i32), ("dtype", _i32), ("batch", _i64), ("heads", _i64), ("rows", _i64), ("width", _i64)]


class SlnFwdArgs(ctypes.Structure):
    _fields_ = _HEAD + [("eps", ctypes.c_float), ("center", _i32), ("weight_dtype", _i32), ("weight_heads", _i32),
                        ("x", TdaTensor), ("y", TdaTensor), ("weight", _p), ("bias", _p), ("stats", _p)]


class SlnBwdArgs(ctypes.Structure):
    _fields_ = _HEAD + [("weight_dtype", _i32), ("weight_heads", _i32), ("center", _i32), ("reserved", _i32),
                        ("x", TdaTensor), ("dy", TdaTensor), ("dx", TdaTensor), ("weight", _p), ("stats", _p),
                        ("dweight", _p), ("dbias", _p), ("workspace", _p), ("workspace_bytes", ctypes.c_size_t)]


# Every function include/sln.h declares: name -> (restype, argtypes)
SIGNATURES = {
    "sln_abi_version": (_i32, []),
    "sln_error_string": (ctypes.c_char_p, [_i32]),
    "sln_bwd_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(SlnBwdArgs)]),
    "sln_validate_fwd": (_i32, [ctypes.POINTER(SlnFwdArgs)]),
    "sln_validate_bwd": (_i32, [ctypes.POINTER(SlnBwdArgs)]),
    "sln_fwd": (_i32, [ctypes.POINTER(SlnFwdArgs), _p]),
    "sln_bwd": (_i32, [ctypes.POINTER(SlnBwdArgs), _p]),
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
        v = lib.sln_abi_version()
        if v != ABI_VERSION:
            raise RuntimeError(f"tda_amd: {_abi.lib_path()} has layer norm ABI version {v}, expected {ABI_VERSION}")
        _lib = lib
    return _lib


def check(code: int, what: str) -> None:
    """Argument errors -> ValueError, launch failures -> TdaError (a RuntimeError)."""
    if code == _abi.OK:
        return
    lib = load()
    msg = f"{what}: {lib.sln_error_string(code).decode()} (code {code})"
    if code == _abi.ERR_HIP:
        raise _abi.TdaError(code, f"{msg}; hipError_t {lib.tda_last_hip_error()}")
    raise ValueError(msg)
