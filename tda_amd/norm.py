"""Layer norm and RMS norm over the last axis, with their gradients: of a head's outputs, as differential attention
wants them, or of whole rows."""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _sln_abi
from .softmax import _CODE, _COMPUTE, _TENSORS, _raw_stream, _refuse_tangents, _row_strides, _sig

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
# where a call's arrays stand in its argument block, in pointers
_FX, _FY, _FW, _FB, _FS = (getattr(_sln_abi.SlnFwdArgs, n).offset // 8 for n in ("x", "y", "weight", "bias", "stats"))
_BX, _BDY, _BDX, _BW, _BS, _BDW, _BDB, _BWS = (getattr(_sln_abi.SlnBwdArgs, n).offset // 8
                                               for n in ("x", "dy", "dx", "weight", "stats", "dweight", "dbias", "workspace"))


def _call(fn, args_type, buf, device, what):
    a = args_type.from_buffer(buf)
    if _current_device() == device.index:
        rc = fn(ctypes.byref(a), _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(ctypes.byref(a), _raw_stream(device.index))
    if rc:
        _sln_abi.check(rc, what)


class _Plan:
    """What a call's signature settles: its argument blocks but for the device pointers, the shape and strides of its
    result.  Rows are (batch, heads, rows, width), axes that x lacks being of one element."""

    __slots__ = ("block", "shape", "strides", "rows", "center", "weight_dtype", "weight_heads", "bwd")

    def __init__(self, x, weight, bias, eps, center):
        w = weight if weight is not None else bias
        self.shape, self.center = x.shape, center
        self.rows = (1,) * (4 - x.dim()) + tuple(x.shape)
        self.strides = _row_strides(x, x.shape[3]) if x.dim() == 4 else torch.empty(x.shape, device="meta").stride()
        self.weight_dtype = _CODE[w.dtype if w is not None else x.dtype]
        self.weight_heads = int(w is not None and w.dim() == 2)
        self.bwd: dict = {}  # argument block and workspace, by what _backward finds
        a = _sln_abi.SlnFwdArgs()
        self.head(a, x)
        a.eps = eps
        a.y.stride[:] = self.four(self.strides)
        self.block = bytes(a)

    def head(self, a, x):
        a.abi_version, a.dtype, a.center = _sln_abi.ABI_VERSION, _CODE[x.dtype], int(self.center)
        a.batch, a.heads, a.rows, a.width = self.rows
        a.weight_dtype, a.weight_heads = self.weight_dtype, self.weight_heads
        a.x.stride[:] = self.four(x.stride())

    def four(self, strides):
        """The strides of four axes.  The last one as it is, for sln_fwd and sln_bwd to check; along one value any will do."""
        return (*(0,) * (4 - len(strides)), *strides[:-1], strides[-1] if self.rows[3] > 1 else 1)

    def backward_block(self, key, x, dy, want):
        a = _sln_abi.SlnBwdArgs()
        self.head(a, x)
        a.dy.stride[:] = self.four(dy.stride())
        if want[0]:
            a.dx.stride[:] = self.four(self.strides)
        a.dweight, a.dbias = (4 if w else None for w in want[1:])
        a.workspace_bytes = _sln_abi.load().sln_bwd_workspace_bytes(ctypes.byref(a))
        if len(self.bwd) > 64:
            self.bwd.clear()
        got = self.bwd[key] = bytes(a), a.workspace_bytes
        return got

    def forward(self, x, weight, bias, stats):
        y = torch.empty_strided(self.shape, self.strides, dtype=x.dtype, device=x.device)
        buf = bytearray(self.block)
        put = memoryview(buf).cast("Q")
        put[_FX], put[_FY] = x.data_ptr(), y.data_ptr()
        if weight is not None:
            put[_FW] = weight.data_ptr()
        if bias is not None:
            put[_FB] = bias.data_ptr()
        if stats is not None:
            put[_FS] = stats.data_ptr()
        _call(_sln_abi.load().sln_fwd, _sln_abi.SlnFwdArgs, buf, x.device, "sln_fwd")
        return y

    def run(self, x, weight, bias):
        if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad
                                        or bias is not None and bias.requires_grad):
            return _LayerNorm.apply(x, weight, bias, self)
        return self.forward(x, weight, bias, None)


_plans: dict = {}  # by signature, of calls whose tensors need no copy: no checks again


def _backward(ctx, dy):
    x, weight, stats = ctx.saved_tensors
    plan, bias = ctx.cfg
    # as they are now: a hook on saved tensors may have brought back copies with other strides
    x, weight, stats = _in_rows(x), None if weight is None else weight.contiguous(), stats.contiguous()
    want = ctx.needs_input_grad[:3]
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    if dy.stride(-1) != 1 and dy.shape[-1] > 1:
        dy = dy.contiguous()
    key = x.stride(), x.dtype, dy.stride(), want
    block, size = plan.bwd.get(key) or plan.backward_block(key, x, dy, want)
    buf = bytearray(block)
    put = memoryview(buf).cast("Q")
    dx = dw = db = None
    if want[0]:
        dx = torch.empty_strided(plan.shape, plan.strides, dtype=x.dtype, device=x.device)
        put[_BDX] = dx.data_ptr()
    if weight is not None:
        put[_BW] = weight.data_ptr()
        if want[1]:
            dw = torch.empty_like(weight)
            put[_BDW] = dw.data_ptr()
    if want[2]:
        db = torch.empty(bias[0], dtype=bias[1], device=x.device)
        put[_BDB] = db.data_ptr()
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        put[_BWS] = ws.data_ptr()
    put[_BX], put[_BDY], put[_BS] = x.data_ptr(), dy.data_ptr(), stats.data_ptr()
    _call(_sln_abi.load().sln_bwd, _sln_abi.SlnBwdArgs, buf, x.device, "sln_bwd")
    return dx, dw, db, None


_backward_once = once_differentiable(_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, plan):
        stats = torch.empty(plan.rows[:3] + (2,), dtype=torch.float32, device=x.device)
        ctx.save_for_backward(x, weight, stats)
        ctx.cfg = plan, None if bias is None else (bias.shape, bias.dtype)
        return plan.forward(x, weight, bias, stats)

    @staticmethod
    def backward(ctx, dy):
        # what refuses a second derivative is set up where one may be taken
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


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


def _in_rows(x):
    """x with up to four axes, and rows that the kernels read in place (x itself or a view where they can), else copied."""
    if x.dim() > 4:
        x = x.flatten(0, -2)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, center=True):
    """(x - mean) / sqrt(var + eps) weight + bias over the last axis; with center=False the mean is left out: x /
    sqrt(mean(x^2) + eps) weight + bias (RMS norm).

    x: float32, bfloat16, float16, or float64 (computed in float32), of any shape, the last axis up to 16384; rows of
    any strides with a unit last one are read in place.  weight, bias: (width,), or (heads, width) with x
    (batch, heads, seq_len, width): each head's own; x's dtype or float32, both alike.  Means and sums are
    float32.  Gradients flow to all three; second derivatives and forward-mode derivatives raise."""
    _refuse_tangents("layer_norm", x, weight, bias)
    eps, center = float(eps), bool(center)  # their values: a plan must not go by which tensor holds them
    key = None
    if type(x) in _TENSORS and (weight is None or type(weight) in _TENSORS) and (bias is None or type(bias) in _TENSORS):
        key = _sig(x), None if weight is None else _sig(weight), None if bias is None else _sig(bias), eps, center
        plan = _plans.get(key)
        if plan is not None:
            return plan.run(x, weight, bias)
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
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if weight is not None:
        _check_weight(weight, "weight", x, None)
    if bias is not None:
        _check_weight(bias, "bias", x, weight)
    if x.dtype == torch.float64:
        return layer_norm(x.float(), *(None if t is None else t.float() for t in (weight, bias)), eps, center=center).double()
    if x.numel() == 0:  # no rows: connected to the inputs
        return x * 1 + sum((t.sum() * 0 for t in (weight, bias) if t is not None), torch.zeros((), device=x.device)).to(x.dtype)
    now = _in_rows(x), None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous()
    plan = _Plan(*now, eps, center)
    if key is not None and all(a is b for a, b in zip(now, (x, weight, bias))):
        if len(_plans) > 4096:
            _plans.clear()
        _plans[key] = plan
    y = plan.run(*now)
    return y if y.shape == x.shape else y.view(x.shape)
