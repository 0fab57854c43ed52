"""ctypes binding of the softmax differential attention operators (include/sda.h) in libtda_hip.so."""
from __future__ import annotations

import ctypes
import threading

from . import _abi
from ._abi import TdaTensor

ABI_VERSION = 1
DTYPE_F16 = 2

ERR_HEADS = -20
ERR_SCALE = -21
ERR_AXES = -22
ERR_CACHE = -23

MAX_AXES = 4
MAX_ROTARY = 4

_i32, _i64, _p = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p

_HEAD = [("abi_version", _i32), ("dtype", _i32), ("causal", _i32), ("scale", ctypes.c_float), ("batch", _i64),
         ("heads", _i64), ("kv_heads", _i64), ("seq_len", _i64), ("seq_len_kv", _i64), ("head_dim", _i64),
         ("v_head_dim", _i64)]
_ROWS = [(n, TdaTensor) for n in ("q1", "k1", "q2", "k2", "v")]
_SIGHT = [("lambda_param", _p), ("lambda_stride", _i64 * 3), ("lambda_dtype", _i32), ("reserved", _i32),
          ("q_offset", _i64), ("q_offsets", _p), ("kv_lens", _p), ("lse", _p)]
_WORK = [("workspace", _p), ("workspace_bytes", ctypes.c_size_t)]


class SdaFwdArgs(ctypes.Structure):
    _fields_ = _HEAD + _ROWS + [("out", TdaTensor), ("out2", TdaTensor), ("out_low", TdaTensor)] + _SIGHT + _WORK


class SdaBwdArgs(ctypes.Structure):
    _fields_ = (_HEAD + _ROWS + [(n, TdaTensor) for n in ("out", "out2", "out_low", "dout", "dq1", "dk1", "dq2", "dk2", "dv")]
                + _SIGHT + [("dlambda", _p)] + _WORK)


class SdaRotaryArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("interleaved", _i32), ("inverse", _i32), ("batch", _i64),
                ("seq_len", _i64), ("head_dim", _i64), ("rot", _i64), ("axes", _i32), ("sections", _i32 * MAX_AXES),
                ("count", _i32), ("heads", _i64 * MAX_ROTARY), ("x", TdaTensor * MAX_ROTARY),
                ("y", TdaTensor * MAX_ROTARY), ("positions", _p), ("position_stride", _i64 * 3),
                ("position_dtype", _i32), ("reserved", _i32), ("inv_freq", _p)]


class SdaKv4(ctypes.Structure):
    _fields_ = [(n, _i64) for n in ("batch", "kv_heads", "capacity", "head_dim", "v_head_dim")] + [
        (n, _p) for n in ("k1", "k2", "v", "lengths")]


_KV = [("abi_version", _i32), ("dtype", _i32), ("cache", SdaKv4)]
_KVROWS = [("rows", _i64), ("k1", TdaTensor), ("k2", TdaTensor), ("v", TdaTensor)]


class SdaKv4AppendArgs(ctypes.Structure):
    _fields_ = _KV + _KVROWS + [("start", _p), ("counts", _p)]


class SdaKv4ReadArgs(ctypes.Structure):
    _fields_ = _KV + _KVROWS


class SdaKv4AttendArgs(ctypes.Structure):
    _fields_ = _KV + [("heads", _i64), ("seq_len", _i64), ("scale", ctypes.c_float), ("lambda_dtype", _i32),
                      ("q1", TdaTensor), ("q2", TdaTensor), ("out", TdaTensor), ("lambda_param", _p),
                      ("lambda_stride", _i64 * 3)] + _WORK


def _call(args):
    return _i32, [ctypes.POINTER(args), _p]


def _on(res, args):
    return res, [ctypes.POINTER(args)]


# Every function include/sda.h declares: name -> (restype, argtypes)
SIGNATURES = {
    "sda_abi_version": (_i32, []),
    "sda_error_string": (ctypes.c_char_p, [_i32]),
    "sda_fwd_workspace_bytes": _on(ctypes.c_size_t, SdaFwdArgs),
    "sda_bwd_workspace_bytes": _on(ctypes.c_size_t, SdaBwdArgs),
    "sda_kv4_attend_workspace_bytes": _on(ctypes.c_size_t, SdaKv4AttendArgs),
    "sda_kv4_bytes": (ctypes.c_size_t, [_i64] * 4),
    "sda_validate_fwd": _on(_i32, SdaFwdArgs),
    "sda_validate_bwd": _on(_i32, SdaBwdArgs),
    "sda_validate_rotary": _on(_i32, SdaRotaryArgs),
    "sda_validate_kv4_append": _on(_i32, SdaKv4AppendArgs),
    "sda_validate_kv4_read": _on(_i32, SdaKv4ReadArgs),
    "sda_validate_kv4_attend": _on(_i32, SdaKv4AttendArgs),
    "sda_fwd": _call(SdaFwdArgs),
    "sda_bwd": _call(SdaBwdArgs),
    "sda_rotary": _call(SdaRotaryArgs),
    "sda_kv4_append": _call(SdaKv4AppendArgs),
    "sda_kv4_read": _call(SdaKv4ReadArgs),
    "sda_kv4_attend": _call(SdaKv4AttendArgs),
}

_lock = threading.Lock()
_lib = None


def load():
    """The library with these functions bound (RuntimeError when it is missing or older)."""
    global _lib
    if _lib is not None:
        return _lib
    lib = _abi.load()
    with _lock:
        for name, (res, args) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError:
                raise RuntimeError(f"tda_amd: {_abi.lib_path()} has no {name}; build it again with "
                                   "`python -m tda_amd.build`") from None
            fn.restype, fn.argtypes = res, args
        v = lib.sda_abi_version()
        if v != ABI_VERSION:
            raise RuntimeError(f"tda_amd: {_abi.lib_path()} has softmax ABI version {v}, expected {ABI_VERSION}")
        _lib = lib
    return _lib


def check(code: int, what: str) -> None:
    """Argument errors -> ValueError, launch failures -> TdaError (a RuntimeError)."""
    if code == _abi.OK:
        return
    lib = load()
    msg = f"{what}: {lib.sda_error_string(code).decode()} (code {code})"
    if code == _abi.ERR_HIP:
        raise _abi.TdaError(code, f"{msg}; hipError_t {lib.tda_last_hip_error()}")
    raise ValueError(msg)
