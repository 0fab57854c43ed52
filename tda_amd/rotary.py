"""Rotary positions with several axes (a token of an image or a video has a row, a column, a time),
applied to the queries and keys before attention, with the gradient.
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _sda_abi, ops
from .softmax import _CODE, _TENSORS, _free_of_grad, _launch, _new_rows, _refuse_tangents, _sig

_PUT = struct.Struct("<Q").pack_into
_OFF = {n: getattr(_sda_abi.SdaRotaryArgs, n).offset for n in ("x", "y", "positions", "inv_freq")}
_TENSOR = ctypes.sizeof(_sda_abi.TdaTensor)


def _readable(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 and t.stride(2) * t.element_size() <= 1 << 25 else t.contiguous()


# Calls without gradients whose tensors are read in place, by signature: their argument block and the outputs'
# strides; such a call takes fresh pointers alone.
_plans: dict = {}


def _block(xs, ys, positions, sections, interleaved: bool, inverse: bool) -> bytes:
    a = _sda_abi.SdaRotaryArgs()
    a.abi_version, a.dtype = _sda_abi.ABI_VERSION, _CODE[xs[0].dtype]
    a.interleaved, a.inverse = int(interleaved), int(inverse)
    a.batch, _, a.seq_len, a.head_dim = xs[0].shape
    a.rot, a.axes, a.count = 2 * sum(sections), len(sections), len(xs)
    a.sections[:len(sections)] = sections
    for i, (x, y) in enumerate(zip(xs, ys)):
        a.heads[i] = x.shape[1]
        a.x[i].stride[:] = x.stride()
        a.y[i].stride[:] = y.stride()
    a.position_stride[:] = positions.stride()
    a.position_dtype = positions.element_size()
    return bytes(a)


def _run(block, xs, ys, positions, inv_freq):
    buf = bytearray(block)
    for i, (x, y) in enumerate(zip(xs, ys)):
        _PUT(buf, _OFF["x"] + i * _TENSOR, x.data_ptr())
        _PUT(buf, _OFF["y"] + i * _TENSOR, y.data_ptr())
    _PUT(buf, _OFF["positions"], positions.data_ptr())
    _PUT(buf, _OFF["inv_freq"], inv_freq.data_ptr())
    _launch(_sda_abi.load().sda_rotary, _sda_abi.SdaRotaryArgs, buf, xs[0].device, "sda_rotary")


def _turn(xs, positions, inv_freq, sections, interleaved: bool, inverse: bool):
    """One sda_rotary launch: new tensors with xs turned (inverse: turned back)."""
    xs = [_readable(x) for x in xs]
    ys = [_new_rows(x, x.shape[3]) for x in xs]
    key = ("sda_rotary", xs[0].dtype, tuple(x.shape for x in xs), tuple(x.stride() for x in xs), positions.dtype,
           positions.stride(), sections, interleaved, inverse)

    block = ops._cached(key, lambda: _block(xs, ys, positions, sections, interleaved, inverse))
    _run(block, xs, ys, positions, inv_freq)
    return tuple(ys)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, inv_freq, sections, interleaved, *xs):
        ctx.save_for_backward(positions, inv_freq)
        ctx.cfg = (sections, interleaved)
        return _turn(xs, positions, inv_freq, sections, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, *dys):
        positions, inv_freq = ctx.saved_tensors
        want = ctx.needs_input_grad[4:]
        grads = iter(_turn([d for d, w in zip(dys, want) if w], positions, inv_freq, *ctx.cfg, True) if any(want) else ())
        return (None,) * 4 + tuple(next(grads) if w else None for w in want)


def rotary_axes(xs, positions, inv_freq, sections, *, interleaved=False):
    """xs with rotary positions of len(sections) axes applied, in one launch.

    xs: a tensor (batch, heads, seq_len, head_dim) or a sequence of up to four (q1, q2, k1, k2), which may
    differ in heads; float32, bfloat16 or float16.  Returns a tensor or a tuple, in xs' dtype.
    positions: int32 or int64, (axes, batch, seq_len), any strides.  inv_freq: float32, one frequency for
    each rotated pair.  sections: how many pairs turn by each axis, in order; pair p of a row turns by
    positions[axis of p] * inv_freq[p].  The 2 len(inv_freq) first values of a row are rotated, the rest
    copied.  A pair is (p, p + len(inv_freq)), with interleaved (2 p, 2 p + 1).  The angle is taken in 64
    bits.  Gradients flow to xs; second derivatives and forward-mode derivatives raise."""
    one = isinstance(xs, torch.Tensor)
    ts = (xs,) if one else tuple(xs)
    _refuse_tangents("rotary_axes", inv_freq, *ts)
    sections = tuple([int(s) for s in sections])
    key = None
    if type(positions) is torch.Tensor and type(inv_freq) is torch.Tensor and all(type(t) in _TENSORS for t in ts):
        key = (tuple([_sig(t) for t in ts]), _sig(positions), _sig(inv_freq), sections, bool(interleaved))
        plan = _plans.get(key)
        if plan is not None and _free_of_grad(inv_freq, *ts):
            ys = tuple([torch.empty_strided(t.shape, st, dtype=t.dtype, device=t.device) for t, st in zip(ts, plan[1])])
            _run(plan[0], ts, ys, positions, inv_freq)
            return ys[0] if one else ys
    if not 1 <= len(ts) <= _sda_abi.MAX_ROTARY:
        raise ValueError(f"rotary_axes takes 1 to {_sda_abi.MAX_ROTARY} tensors, got {len(ts)}")
    ref = ts[0]
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError("xs must be a torch.Tensor or a sequence of them")
        if t.dim() != 4:
            raise ValueError(f"xs must have shape (batch, heads, seq_len, head_dim), got {tuple(t.shape)}")
        if (t.shape[0], t.shape[2], t.shape[3]) != (ref.shape[0], ref.shape[2], ref.shape[3]):
            raise ValueError(f"xs may differ in heads only, got {tuple(ref.shape)} and {tuple(t.shape)}")
        if t.dtype != ref.dtype or t.device != ref.device:
            raise ValueError("xs must have one dtype and one device")
    dev = ref.device
    if dev.type != "cuda":
        raise ValueError(f"tda_amd runs on the GPU only (HIP); got tensors on {dev}")
    if ref.dtype not in _CODE:
        raise ValueError(f"xs must be float32, bfloat16 or float16, got {ref.dtype}")
    if not 1 <= len(sections) <= _sda_abi.MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must be 1 to {_sda_abi.MAX_AXES} counts of pairs, got {sections}")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a 1-D float32 tensor")
    if inv_freq.requires_grad:
        raise ValueError("inv_freq gets no gradient: detach it")
    pairs = inv_freq.shape[0]
    if pairs < 1 or sum(sections) != pairs or 2 * pairs > ref.shape[3]:
        raise ValueError(f"sections {sections} must add up to inv_freq's {pairs} pairs, at most half of head_dim {ref.shape[3]}")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be an int32 or int64 tensor")
    if positions.shape != (len(sections), ref.shape[0], ref.shape[2]):
        raise ValueError(f"positions must have shape {(len(sections), ref.shape[0], ref.shape[2])}, got {tuple(positions.shape)}")
    if positions.device != dev or inv_freq.device != dev:
        raise ValueError(f"positions and inv_freq must be on {dev}")
    if any(t.shape[1] == 0 for t in ts) or ref.shape[0] == 0 or ref.shape[2] == 0:
        if any(t.numel() for t in ts):
            raise ValueError("a tensor of xs has no heads")
        res = tuple(t.clone() for t in ts)
        return res[0] if one else res
    frequencies, inv_freq = inv_freq, inv_freq.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        res = _Rotary.apply(positions, inv_freq, sections, bool(interleaved), *ts)
    else:
        res = _turn(ts, positions, inv_freq, sections, bool(interleaved), False)
        if key is not None and inv_freq is frequencies and all(_readable(t) is t for t in ts):
            if len(_plans) > 4096:
                _plans.clear()
            _plans[key] = _block(ts, res, positions, sections, bool(interleaved), False), [y.stride() for y in res]
    return res[0] if one else res
