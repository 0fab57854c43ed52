"""Layer norm and RMS norm over the last axis, with their gradients: of a head's outputs, as differential attention
wants them, or of whole rows."""
from __future__ import annotations

import ctypes
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _sln_abi, ops
from .softmax import _CODE, _COMPUTE, _TENSORS, _free_of_grad, _new_rows, _raw_stream, _refuse_tangents, _sig

_PUT = struct.Struct("<Q").pack_into
_FWD_OFF = {n: getattr(_sln_abi.SlnFwdArgs, n).offset for n in ("x", "y", "weight", "bias", "stats")}
_BWD_OFF = {n: getattr(_sln_abi.SlnBwdArgs, n).offset for n in ("x", "dy", "dx", "weight", "stats", "dweight", "dbias", "workspace")}

_plans: dict = {}  # of calls without gradients whose tensors need no copy, by signature: no checks again


def _readable(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _strides(t: torch.Tensor):
    return (*t.stride()[:3], 1)


def _rows4(x: torch.Tensor) -> torch.Tensor:
    """x as (batch, heads, rows, width), a view where its strides allow one."""
    if x.dim() == 4:
        return x
    if x.dim() == 3:
        return x.unsqueeze(1)
    return x.reshape(1, 1, -1, x.shape[-1])


def _call(fn, args_type, buf, device, what):
    a = args_type.from_buffer(buf)
    if torch.cuda.current_device() == device.index:
        rc = fn(ctypes.byref(a), _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(ctypes.byref(a), _raw_stream(device.index))
    if rc:
        _sln_abi.check(rc, what)


def _head(a, x, weight, bias, center):
    w = weight if weight is not None else bias
    a.abi_version, a.dtype, a.center = _sln_abi.ABI_VERSION, _CODE[x.dtype], int(center)
    a.batch, a.heads, a.rows, a.width = x.shape
    a.weight_dtype = _CODE[w.dtype if w is not None else x.dtype]
    a.weight_heads = int(w is not None and w.dim() == 2)
    a.x.stride[:] = _strides(x)


def _fwd_block(x, y, weight, bias, eps, center) -> bytes:
    a = _sln_abi.SlnFwdArgs()
    _head(a, x, weight, bias, center)
    a.eps = eps
    a.y.stride[:] = _strides(y)
    return bytes(a)


def _forward(block, x, y, weight, bias, stats):
    buf = bytearray(block)
    for name, t in (("x", x), ("y", y), ("weight", weight), ("bias", bias), ("stats", stats)):
        if t is not None:
            _PUT(buf, _FWD_OFF[name], t.data_ptr())
    _call(_sln_abi.load().sln_fwd, _sln_abi.SlnFwdArgs, buf, x.device, "sln_fwd")


def _key(kind, rows, weight, bias, *more):
    return (kind, rows[0].shape, rows[0].dtype, tuple([None if t is None else t.stride() for t in rows]),
            tuple([None if t is None else (t.dtype, t.dim()) for t in (weight, bias)]), *more)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, center):
        x = _readable(x)
        y = _new_rows(x, x.shape[3])
        stats = torch.empty(x.shape[:3] + (2,), dtype=torch.float32, device=x.device)
        block = ops._cached(_key("sln_fwd", (x, y), weight, bias, eps, center), lambda: _fwd_block(x, y, weight, bias, eps, center))
        _forward(block, x, y, weight, bias, stats)
        ctx.save_for_backward(x, weight, stats)
        ctx.cfg = (None if bias is None else (bias.shape, bias.dtype), center)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        like_bias, center = ctx.cfg
        dy = _readable(dy if dy.dtype == x.dtype else dy.to(x.dtype))
        want = ctx.needs_input_grad
        dx = _new_rows(x, x.shape[3]) if want[0] else None
        dw = torch.empty_like(weight) if want[1] else None
        db = torch.empty(like_bias[0], dtype=like_bias[1], device=x.device) if want[2] else None

        def build():
            a = _sln_abi.SlnBwdArgs()
            _head(a, x, weight, db, center)
            a.dy.stride[:] = _strides(dy)
            if dx is not None:
                a.dx.stride[:] = _strides(dx)
            a.dweight, a.dbias = (None if t is None else 4 for t in (dw, db))
            a.workspace_bytes = _sln_abi.load().sln_bwd_workspace_bytes(ctypes.byref(a))
            return bytes(a), a.workspace_bytes

        block, size = ops._cached(_key("sln_bwd", (x, dy, dx), weight, db, center, want[:3]), build)
        buf = bytearray(block)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        for name, t in (("x", x), ("dy", dy), ("dx", dx), ("weight", weight), ("stats", stats), ("dweight", dw), ("dbias", db),
                        ("workspace", ws)):
            if t is not None:
                _PUT(buf, _BWD_OFF[name], t.data_ptr())
        _call(_sln_abi.load().sln_bwd, _sln_abi.SlnBwdArgs, buf, x.device, "sln_bwd")
        return dx, dw, db, None, None


def _check_weight(w, name, x, other):
    if not isinstance(w, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if w.device != x.device:
        raise ValueError(f"device mismatch: x {x.device} vs {name} {w.device}")
    if w.shape != x.shape[-1:] and not (x.dim() == 4 and w.shape == (x.shape[1], x.shape[3])):
        raise ValueError(f"{name} must have shape ({x.shape[-1]},)" + (f" or {(x.shape[1], x.shape[3])}" if x.dim() == 4 else "")
                         + f", got {tuple(w.shape)}")
    if w.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    if other is not None and (other.shape != w.shape or other.dtype != w.dtype):
        raise ValueError(f"weight and bias must be alike, got {tuple(other.shape)} {other.dtype} and {tuple(w.shape)} {w.dtype}")


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, center=True):
    """(x - mean) / sqrt(var + eps) weight + bias over the last axis; with center=False the mean is left out: x /
    sqrt(mean(x^2) + eps) weight + bias (RMS norm).

    x: float32, bfloat16, float16, or float64 (computed in float32), of any shape, the last axis up to 16384; rows of
    any strides with a unit last one are read in place.  weight, bias: (width,), or (heads, width) with x
    (batch, heads, seq_len, width): each head's own; x's dtype or float32, both alike.  Means and sums are
    float32.  Gradients flow to all three; second derivatives and forward-mode derivatives raise."""
    _refuse_tangents("layer_norm", x, weight, bias)
    key = None
    if type(x) in _TENSORS and (weight is None or type(weight) in _TENSORS) and (bias is None or type(bias) in _TENSORS):
        key = _sig(x), None if weight is None else _sig(weight), None if bias is None else _sig(bias), eps, bool(center)
        plan = _plans.get(key)
        if plan is not None and _free_of_grad(*[t for t in (x, weight, bias) if t is not None]):
            y = torch.empty_strided(plan[1], plan[2], dtype=x.dtype, device=x.device)
            _forward(plan[0], x, y, weight, bias, None)
            return y
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.dim() < 1:
        raise ValueError("x must have an axis")
    if x.device.type != "cuda":
        raise ValueError(f"tda_amd runs on the GPU only (HIP); got tensors on {x.device}")
    if x.dtype not in _COMPUTE:
        raise ValueError(f"x must be float32, bfloat16, float16 or float64, got {x.dtype}")
    if not 1 <= x.shape[-1] <= _sln_abi.MAX_WIDTH:
        raise ValueError(f"the last axis must have 1 to {_sln_abi.MAX_WIDTH} values, got {x.shape[-1]}")
    e = float(eps)
    if not (e >= 0 and math.isfinite(e)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if weight is not None:
        _check_weight(weight, "weight", x, None)
    if bias is not None:
        _check_weight(bias, "bias", x, weight)
    given = x, weight, bias
    if x.dtype == torch.float64:
        x, weight, bias = (None if t is None else t.to(torch.float32) for t in given)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    if x.numel() == 0:
        return x * 1 + sum((t.sum() * 0 for t in (weight, bias) if t is not None), torch.zeros((), dtype=x.dtype, device=x.device)).to(x.dtype)
    rows = _rows4(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        y = _LayerNorm.apply(rows, weight, bias, e, bool(center))
    else:
        r = _readable(rows)
        y = _new_rows(r, r.shape[3])
        block = _fwd_block(r, y, weight, bias, e, bool(center))
        _forward(block, r, y, weight, bias, None)
        if key is not None and r is rows and x is given[0] and weight is given[1] and bias is given[2] and rows.data_ptr() == x.data_ptr():
            if len(_plans) > 4096:
                _plans.clear()
            out = y.view(x.shape) if x.dim() != 4 else y
            _plans[key] = block, out.shape, out.stride()
    if y.shape != x.shape:
        y = y.view(x.shape)
    return y if y.dtype == given[0].dtype else y.to(given[0].dtype)
