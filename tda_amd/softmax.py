"""Softmax differential attention: the difference of two softmax maps with a learned weight,

    out = (softmax(s q1 k1^T + M) - lambda softmax(s q2 k2^T + M)) v

beside the threshold form of api.py.  Forward and backward run in hand-written kernels behind
include/sda.h (float32, bfloat16, float16; float64 is computed in float32, as by the threshold
operators); a call of few query rows, such as a decoding step, takes kernels that split the key axis.
There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _abi, _sda_abi, ops

_PUT = struct.Struct("<Q").pack_into
_COMPUTE = {torch.float32: torch.float32, torch.bfloat16: torch.bfloat16,
            torch.float16: torch.float16, torch.float64: torch.float32}
_CODE = {torch.float32: _abi.DTYPE_F32, torch.bfloat16: _abi.DTYPE_BF16, torch.float16: _sda_abi.DTYPE_F16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)  # the current stream's handle
_ROW_BYTES = 1 << 25  # the largest distance between rows that the kernels take

_FWD_ROWS = ("q1", "k1", "q2", "k2", "v", "out", "out2", "out_low")
_BWD_ROWS = ("q1", "k1", "q2", "k2", "v", "out", "out2", "out_low", "dout", "dq1", "dk1", "dq2", "dk2", "dv")


def _offsets(args, names):
    return {n: getattr(args, n).offset for n in names}


_TENSORS = (torch.Tensor, torch.nn.Parameter)
_FWD_OFF = _offsets(_sda_abi.SdaFwdArgs, _FWD_ROWS + ("lambda_param", "q_offsets", "kv_lens", "lse", "workspace"))
_PLAN_OFF = [_FWD_OFF[n] for n in ("q1", "q2", "k1", "k2", "v")]
_BWD_OFF = _offsets(_sda_abi.SdaBwdArgs, _BWD_ROWS + ("lambda_param", "q_offsets", "kv_lens", "lse", "dlambda", "workspace"))


# ------------------------------------------------------------------ arguments
_stride_ok: dict = {}  # (strides, element size): whether rows laid out so can be read in place


def _usable(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place, else a contiguous copy."""
    st, es = t.stride(), t.element_size()
    ok = _stride_ok.get((st, es))
    if ok is None:
        if len(_stride_ok) > 4096:
            _stride_ok.clear()
        ok = _stride_ok[st, es] = (st[3] == 1 and all(s >= 0 and s * es % 16 == 0 for s in st[:3])
                                   and st[2] * es <= _ROW_BYTES)
    return t if ok and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _apart(t: torch.Tensor) -> torch.Tensor:
    """t itself, or a contiguous copy where its rows overlap (a stride of 0 along the sequence, as that of the gradient
    of a sum or mean over it) and sda_bwd does not take them so."""
    n, width = t.shape[2:]
    return t.clone(memory_format=torch.contiguous_format) if n % 32 and t.stride(2) < width else t


def _check_rows(tensors, names, shapes=None):
    """4-D floating tensors of one dtype on one GPU, the batch the same."""
    ref = tensors[0]
    dtype, device = getattr(ref, "dtype", None), getattr(ref, "device", None)
    for t, n in zip(tensors, names):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{n} must be a torch.Tensor")
        if t.dim() != 4:
            raise ValueError(f"{n} must have shape (batch, heads, seq_len, head_dim), got {tuple(t.shape)}")
        if t.dtype != dtype:
            raise ValueError(f"dtype mismatch: {names[0]} {dtype} vs {n} {t.dtype}")
        if t.device != device:
            raise ValueError(f"device mismatch: {names[0]} {device} vs {n} {t.device}")
    if ref.device.type != "cuda":
        raise ValueError(f"tda_amd runs on the GPU only (HIP); got tensors on {ref.device}")
    if not ref.dtype.is_floating_point:
        raise ValueError(f"floating-point inputs required, got {ref.dtype}")


def _check_heads(heads: int, kv_heads: int):
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of the key/value heads ({kv_heads})")


def _scale(scale, d: int) -> float:
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 1e-30 <= s <= 1e30:  # s log2(e) and its reciprocal stay in 32 bits
        raise ValueError(f"scale must be finite and positive (1e-30 to 1e30), got {s}")
    return s


def _lambda(lam, b: int, h: int, n: int, device) -> torch.Tensor:
    """lambda_param as a device tensor of a kernel dtype: a scalar, (heads,) or something that
    broadcasts to (batch, heads, seq_len)."""
    if not isinstance(lam, torch.Tensor):
        return torch.full((), float(lam), dtype=torch.float32, device=device)
    if lam.numel() != 1 and not (lam.dim() == 1 and lam.shape[0] == h) and not (
            lam.dim() == 3 and all(x in (1, y) for x, y in zip(lam.shape, (b, h, n)))):
        raise ValueError(f"lambda_param must be a scalar, ({h},) or broadcast to ({b}, {h}, {n}), got {tuple(lam.shape)}")
    if not lam.dtype.is_floating_point:
        raise ValueError(f"lambda_param must be floating-point, got {lam.dtype}")
    if lam.device != device or lam.dtype not in _CODE:
        lam = lam.to(device=device, dtype=lam.dtype if lam.dtype in _CODE else torch.float32)
    return lam


def _lambda_strides(lam: torch.Tensor):
    """(b, h, i) element strides; 0 along an axis of one element.  lam holds an element of its own
    for every index (_own)."""
    if lam.numel() == 1:
        return 0, 0, 0
    if lam.dim() == 1:
        return 0, lam.stride(0), 0
    return tuple(0 if n == 1 else s for n, s in zip(lam.shape, lam.stride()))


def _own(lam: torch.Tensor) -> torch.Tensor:
    """lam with no two indices at one place (an expanded tensor's gradient has an element for each)."""
    return lam.contiguous() if any(n > 1 and s == 0 for n, s in zip(lam.shape, lam.stride())) else lam


def _ints(x, b: int, device, name: str) -> torch.Tensor:
    """A (batch,) int32 tensor on the device."""
    if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.shape[0] != b:
        raise ValueError(f"{name} must be a tensor of shape ({b},)")
    if x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must hold int32 or int64, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, got {x.device}")
    if x.dtype == torch.int64:  # a value beyond 32 bits keeps its sign and its side
        x = x.clamp(-(1 << 30), 1 << 30)
    return x.to(torch.int32).contiguous()


def _dims(d: int, dv: int):
    """The kernels' (head_dim, v_head_dim) for a caller's, whose rows are padded with zeros."""
    for kd, kv in ((64, 64), (64, 128), (128, 128), (128, 256)):
        if d <= kd and dv <= kv:
            return kd, kv
    raise ValueError(f"head_dim must be at most 128 and the values' at most 256, got {d} and {dv}")


def _pad(t: torch.Tensor, d: int) -> torch.Tensor:
    return t if t.shape[-1] == d else F.pad(t, (0, d - t.shape[-1]))


def _row_strides(like: torch.Tensor, width: int):
    """Strides of dense (B, H, N, width) rows in like's memory order."""
    h, n = max(like.shape[1], 1), max(like.shape[2], 1)
    if h > 1 and n > 1 and like.stride(1) < like.stride(2):
        return h * n * width, width, h * width, 1
    return h * n * width, n * width, width, 1


def _new_rows(like: torch.Tensor, width: int, dtype=None) -> torch.Tensor:
    """Uninitialised (B, H, N, width) rows in like's memory order."""
    return torch.empty_strided((*like.shape[:3], width), _row_strides(like, width), dtype=dtype or like.dtype, device=like.device)


# ------------------------------------------------------------------ calls
def _template(kind, rows, names, args_type, size_fn, lam, scale, causal, q_offset, more=()):
    """(template bytes, workspace bytes) of a call: every field but the device pointers, cached by
    what they depend on."""
    q, k, v = rows[0], rows[1], rows[4]
    ls = _lambda_strides(lam)
    key = (kind, q.shape, k.shape, v.shape, q.dtype, lam.dtype, ls, scale, causal, q_offset, more,
           tuple(None if t is None else t.stride() for t in rows))

    def build():
        a = args_type()
        a.abi_version, a.dtype, a.causal, a.scale = _sda_abi.ABI_VERSION, _CODE[q.dtype], int(causal), scale
        a.batch, a.heads, a.seq_len, a.head_dim = q.shape
        a.kv_heads, a.seq_len_kv, a.v_head_dim = v.shape[1], v.shape[2], v.shape[3]
        for name, t in zip(names, rows):
            if t is not None:
                getattr(a, name).stride[:] = t.stride()
                getattr(a, name).data = 1  # present; the call's own pointer replaces it
        a.lambda_stride[:] = ls
        a.lambda_dtype = _CODE[lam.dtype]
        a.q_offset = q_offset
        if kind == "sda_fwd":
            a.lse = 1 if more[0] else None
        size = getattr(_sda_abi.load(), size_fn)(ctypes.byref(a))
        a.workspace_bytes = size
        return bytes(a), size

    return ops._cached(key, build)


# A call whose tensors need no copy and no gradient depends on nothing but their layouts: once such a call
# has passed the checks below, calls of the same signature reuse its argument block and take fresh pointers alone.
_plans: dict = {}


def _sig(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype, t.device


def _free_of_grad(*tensors) -> bool:
    return not torch.is_grad_enabled() or not any(t.requires_grad for t in tensors)


def _refuse_tangents(what: str, *tensors):
    """A forward-mode derivative is refused, not dropped: a dual tensor need not require a gradient, so the calls that
    leave the autograd function out would return it without its tangent."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no level is open
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


def _plan_key(rows, lam, scale, causal, q_offset, kv_lens):
    """The signature of a forward call that may have a plan, or None."""
    if type(lam) not in _TENSORS or not (q_offset is None or type(q_offset) is int) or not (scale is None or type(scale) is float):
        return None
    for t in rows:
        if type(t) not in _TENSORS:
            return None
    if kv_lens is not None and type(kv_lens) is not torch.Tensor:
        return None
    q1, q2, k1, k2, v = rows
    return (_sig(q1), _sig(q2), _sig(k1), _sig(k2), _sig(v), _sig(lam), scale, bool(causal), q_offset,
            None if kv_lens is None else _sig(kv_lens))


def _run_plan(plan, rows, lam, kv_lens):
    """The planned call's output, or None where a tensor's address does not suit the kernels."""
    tpl, size, shape, strides = plan
    ptrs = [t.data_ptr() for t in rows]
    for p in ptrs:
        if p % 16:
            return None
    q1 = rows[0]
    buf = bytearray(tpl)
    out = torch.empty_strided(shape, strides, dtype=q1.dtype, device=q1.device)
    for at, p in zip(_PLAN_OFF, ptrs):
        _PUT(buf, at, p)
    _PUT(buf, _FWD_OFF["out"], out.data_ptr())
    _PUT(buf, _FWD_OFF["lambda_param"], lam.data_ptr())
    if kv_lens is not None:
        _PUT(buf, _FWD_OFF["kv_lens"], kv_lens.data_ptr())
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=q1.device)
        _PUT(buf, _FWD_OFF["workspace"], ws.data_ptr())
    _launch(_sda_abi.load().sda_fwd, _sda_abi.SdaFwdArgs, buf, q1.device, "sda_fwd")
    return out


def _launch(fn, args_type, buf, device, what):
    a = args_type.from_buffer(buf)
    if torch.cuda.current_device() == device.index:
        rc = fn(ctypes.byref(a), _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(ctypes.byref(a), _raw_stream(device.index))
    if rc:
        _sda_abi.check(rc, what)


def _fill(buf, off, names, tensors):
    for name, t in zip(names, tensors):
        if t is not None:
            _PUT(buf, off[name], t.data_ptr())


def _forward(q1, q2, k1, k2, v, lam, scale, causal, q_offset, q_offsets, kv_lens, saving):
    """One sda_fwd call on usable tensors: out, and (saving) out2, out_low and lse for the backward."""
    lib = _sda_abi.load()
    out = _new_rows(q1, v.shape[3])
    out2 = low = lse = None
    if saving:
        out2 = _new_rows(q1, v.shape[3], torch.float32)
        low = _new_rows(q1, v.shape[3]) if q1.dtype != torch.float32 else None
        lse = torch.empty((2,) + q1.shape[:3], dtype=torch.float32, device=q1.device)
    rows = (q1, k1, q2, k2, v, out, out2, low)
    tpl, size = _template("sda_fwd", rows, _FWD_ROWS, _sda_abi.SdaFwdArgs, "sda_fwd_workspace_bytes", lam, scale,
                          causal, q_offset, (saving,))
    buf = bytearray(tpl)
    _fill(buf, _FWD_OFF, _FWD_ROWS, rows)
    ws = torch.empty(size, dtype=torch.uint8, device=q1.device) if size else None
    _fill(buf, _FWD_OFF, ("lambda_param", "q_offsets", "kv_lens", "lse", "workspace"), (lam, q_offsets, kv_lens, lse, ws))
    _launch(lib.sda_fwd, _sda_abi.SdaFwdArgs, buf, q1.device, "sda_fwd")
    return out, out2, low, lse


class _DifferentialAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q1, q2, k1, k2, v, lam, scale, causal, q_offset, q_offsets, kv_lens):
        saving = any(ctx.needs_input_grad[:6])
        rows = [_usable(t) for t in (q1, q2, k1, k2, v)]
        if saving:
            rows[:2] = _apart(rows[0]), _apart(rows[1])
        out, out2, low, lse = _forward(*rows, lam, scale, causal, q_offset, q_offsets, kv_lens, saving)
        if saving:
            ctx.save_for_backward(*rows, lam, out, out2, low, lse, q_offsets, kv_lens)
            ctx.cfg = (scale, causal, q_offset)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q1, q2, k1, k2, v, lam, out, out2, low, lse, q_offsets, kv_lens = ctx.saved_tensors
        scale, causal, q_offset = ctx.cfg
        lib = _sda_abi.load()
        dout = _apart(_usable(dout if dout.dtype == q1.dtype else dout.to(q1.dtype)))
        dq1, dq2 = _new_rows(q1, q1.shape[3]), _new_rows(q2, q2.shape[3])
        dk1, dk2, dv = (_new_rows(t, t.shape[3]) for t in (k1, k2, v))
        dlam = torch.empty(lam.shape, dtype=lam.dtype, device=lam.device) if ctx.needs_input_grad[5] else None
        rows = (q1, k1, q2, k2, v, out, out2, low, dout, dq1, dk1, dq2, dk2, dv)
        tpl, size = _template("sda_bwd", rows, _BWD_ROWS, _sda_abi.SdaBwdArgs, "sda_bwd_workspace_bytes", lam, scale,
                              causal, q_offset)
        buf = bytearray(tpl)
        _fill(buf, _BWD_OFF, _BWD_ROWS, rows)
        ws = torch.empty(size, dtype=torch.uint8, device=q1.device)
        _fill(buf, _BWD_OFF, ("lambda_param", "q_offsets", "kv_lens", "lse", "dlambda", "workspace"),
              (lam, q_offsets, kv_lens, lse, dlam, ws))
        _launch(lib.sda_bwd, _sda_abi.SdaBwdArgs, buf, q1.device, "sda_bwd")
        grads = (dq1, dq2, dk1, dk2, dv, dlam)
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None,) * 5


def differential_attention(q1, q2, k1, k2, v, lambda_param, scale=None, causal=True, *, q_offset=None, kv_lens=None):
    """(softmax(scale q1 k1^T + M) - lambda_param softmax(scale q2 k2^T + M)) v, by one fused kernel.

    q1, q2: (batch, heads, seq_len, head_dim); k1, k2: (batch, kv_heads, seq_len_kv, head_dim);
    v: (batch, kv_heads, seq_len_kv, v_head_dim), heads a multiple of kv_heads: query head h reads
    key head h // (heads // kv_heads).  Returns (batch, heads, seq_len, v_head_dim) in v's dtype.
    head_dim up to 128 and v_head_dim up to 256; (64, 64), (64, 128), (128, 128) and (128, 256) run in
    place, others are padded with zeros.

    lambda_param: a float, or a tensor that is a scalar, (heads,) or broadcasts to (batch, heads,
    seq_len); unclamped, differentiable.  scale: default 1 / sqrt(head_dim); 1e-30 to 1e30, with scores
    scale q k of up to 1e9 (32 bits hold them to 2^-24).

    M: row i of sequence b stands at position q_offset + i (q_offset an int, by default
    max(seq_len_kv - seq_len, 0), or an int32/int64 tensor (batch,), which may be negative).  With
    causal it sees the keys up to its position; with kv_lens (int32/int64, (batch,), clamped to [0,
    seq_len_kv]) only the first kv_lens[b].  A row that sees no key is zero, with zero gradients, and
    keys that no row of the call sees may hold anything.  (A NaN or infinite value row reaches the rows
    that see it, and may reach other rows of the same call that stand before it.)

    Gradients flow to every tensor; second derivatives and forward-mode derivatives raise."""
    tensors, names = (q1, q2, k1, k2, v), ("q1", "q2", "k1", "k2", "v")
    _refuse_tangents("differential_attention", *tensors, lambda_param)
    key = _plan_key(tensors, lambda_param, scale, causal, q_offset, kv_lens)
    plan = _plans.get(key) if key is not None else None
    if plan is not None and _free_of_grad(*tensors, lambda_param):
        out = _run_plan(plan, tensors, lambda_param, kv_lens)
        if out is not None:
            return out
    _check_rows(tensors, names)
    if q2.shape != q1.shape:
        raise ValueError(f"shape mismatch: q1 {tuple(q1.shape)} vs q2 {tuple(q2.shape)}")
    b, h, n, d = q1.shape
    hk, nk, dv = v.shape[1:]
    for t, name in ((k1, "k1"), (k2, "k2")):
        if t.shape != (b, hk, nk, d):
            raise ValueError(f"shape mismatch: {name} {tuple(t.shape)} must be {(b, hk, nk, d)}")
    if v.shape[0] != b:
        raise ValueError(f"shape mismatch: v {tuple(v.shape)} has another batch than q1 {tuple(q1.shape)}")
    _check_heads(h, hk)
    dev, cdt = q1.device, _COMPUTE.get(q1.dtype)
    if cdt is None:
        raise ValueError(f"unsupported dtype {q1.dtype}")
    s = _scale(scale, max(d, 1))
    kd, kv = _dims(d, dv)
    lam = _own(_lambda(lambda_param, b, h, n, dev))
    q_offsets = None
    if isinstance(q_offset, torch.Tensor) and q_offset.dim():
        q_offsets, off = _ints(q_offset, b, dev, "q_offset"), 0
    else:
        off = _offset(q_offset, n, nk)
    lens = None if kv_lens is None else _ints(kv_lens, b, dev, "kv_lens")
    if any(t.numel() == 0 for t in tensors):  # no rows or no keys: zeros, connected to the inputs
        none = sum(t[:0].sum() for t in tensors) + lam.reshape(-1)[:0].sum().to(q1.dtype)
        return torch.zeros((b, h, n, dv), dtype=q1.dtype, device=dev) + none
    rows = [t if t.dtype == cdt else t.to(cdt) for t in tensors]
    rows = [_pad(t, kd) for t in rows[:4]] + [_pad(rows[4], kv)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in (*rows, lam)):
        out = _DifferentialAttention.apply(*rows, lam, s, bool(causal), off, q_offsets, lens)
    else:
        given = rows
        rows = [_usable(t) for t in rows]
        out = _forward(*rows, lam, s, bool(causal), off, q_offsets, lens, False)[0]
        if key is not None and lam is lambda_param and lens is kv_lens and all(
                a is b is c for a, b, c in zip(rows, given, tensors)):
            if len(_plans) > 4096:
                _plans.clear()
            tpl, size = _template("sda_fwd", (q1, k1, q2, k2, v, out, None, None), _FWD_ROWS, _sda_abi.SdaFwdArgs,
                                  "sda_fwd_workspace_bytes", lam, s, bool(causal), off, (False,))
            _plans[key] = tpl, size, out.shape, out.stride()
    if kv != dv:
        out = out[..., :dv]
    return out if out.dtype == q1.dtype else out.to(q1.dtype)


def _offset(q_offset, n: int, nk: int) -> int:
    """Position of query row 0 (default: the rows are the keys' last positions)."""
    if q_offset is None:
        return max(nk - n, 0)
    off = int(q_offset)
    if off < 0:
        raise ValueError(f"q_offset must be >= 0, got {off}")
    return off
