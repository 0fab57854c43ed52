"""A key/value cache of softmax differential attention held in 4 bits, and the attention over it."""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _sda_abi
from .softmax import (_CODE, _TENSORS, _check_heads, _check_rows, _ints, _lambda, _lambda_strides, _launch, _new_rows, _scale, _sig,
                       _usable, differential_attention)

_PUT = struct.Struct("<Q").pack_into
_DIMS = ((64, 64), (64, 128), (128, 128), (128, 256))
_LENGTHS = _sda_abi.SdaKv4AttendArgs.cache.offset + _sda_abi.SdaKv4.lengths.offset  # the same in all three calls
_ATTEND_OFF = {n: getattr(_sda_abi.SdaKv4AttendArgs, n).offset for n in ("q1", "q2", "out", "lambda_param", "workspace")}
_APPEND_OFF = {n: getattr(_sda_abi.SdaKv4AppendArgs, n).offset for n in ("k1", "k2", "v", "start", "counts")}
_READ_OFF = {n: getattr(_sda_abi.SdaKv4ReadArgs, n).offset for n in ("k1", "k2", "v")}


def _from_codes(batch: int, kv_heads: int, rows: int, dtype) -> bool:
    """Whether attend() computes `rows` query rows for each key head from the codes, 16 rows a pass over them, or
    reads the rows out first, for the attention that passes over them once per 128.  us, codes : rows, (batch, heads, kv_heads, n, keys) of width 128, bf16:
    (8, 16, 4, 16, 4096) 38 : 108, (32, 32, 8, 32, 4096) 344 : 767, (16, 8, 8, 128, 4096) 178 : 238,
    (16, 8, 8, 256, 4096) 331 : 261, (1, 16, 4, 256, 4096) 60 : 94, (1, 16, 4, 512, 4096) 92 : 96; float32:
    (8, 8, 8, 128, 4096) 255 : 1257.  All with full caches: rows are read out for the whole capacity, which takes its time
    and capacity (2 head_dim + v_head_dim) values a key head whatever is held: bf16 prompts of 512 rows into empty caches,
    (32, 32, 8, 512) of capacity 8192 992 : 603, (8, 16, 16, 512) of 8192 and width 64 72 : 121, (1, 32, 8, 512) of 32768
    40 : 58."""
    return rows <= (512 if dtype == torch.float32 else 128) or batch * kv_heads * -(-rows // 16) <= 256


class Int4KVCache:
    """The k1, k2 and v rows of up to `capacity` positions for each of `batch` sequences, 4.5 bits a value.

    Every row is held in groups of 64 values x as m = bf16(min x), s = bf16((max x - m) / 15) (in 32
    bits) and codes rint((x - m) / s) in 0 .. 15 (ties to even; all 0 when s < 2^-100); it stands for m + s
    code.  A group with a NaN or an infinity reads as NaN.  (head_dim, v_head_dim): (64, 64), (64, 128), (128, 128) or (128, 256).  capacity is at most 2^24.

    `lengths` (int32, (batch,), on the device) counts the rows each sequence holds; the calls read and
    write it on the GPU, without synchronising, so they can be captured into a graph.  A program may set
    it, to drop rows or to hand a place to another sequence.  The cache carries no gradient.  copy.deepcopy and
    pickling give a cache with rows and lengths of its own."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, v_head_dim: int | None = None, *,
                 device="cuda"):
        v_head_dim = head_dim if v_head_dim is None else v_head_dim
        for name, n in (("batch", batch), ("kv_heads", kv_heads), ("capacity", capacity)):
            if n < 1:
                raise ValueError(f"{name} must be at least 1, got {n}")
        if (head_dim, v_head_dim) not in _DIMS:
            raise ValueError(f"(head_dim, v_head_dim) must be one of {_DIMS}, got {(head_dim, v_head_dim)}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"tda_amd runs on the GPU only (HIP); got {device}")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.batch, self.kv_heads, self.capacity = int(batch), int(kv_heads), int(capacity)
        self.head_dim, self.v_head_dim, self.device = int(head_dim), int(v_head_dim), device
        lib = _sda_abi.load()
        sizes = [lib.sda_kv4_bytes(batch, kv_heads, capacity, w) for w in (head_dim, head_dim, v_head_dim)]
        if not all(sizes):
            raise ValueError(f"capacity must be at most 2^24 and batch kv_heads below 2^30, got {batch}, {kv_heads}, {capacity}")
        self._held = [torch.empty(n, dtype=torch.uint8, device=device) for n in sizes]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._wide = False          # rows of a wider range than float16's were appended
        self._templates: dict = {}  # argument blocks by configuration
        self._plans: dict = {}      # of calls whose tensors need no copy, by their signature: no checks again

    def __getstate__(self):
        return {**self.__dict__, "_templates": {}, "_plans": {}}  # a copy has buffers of its own: their addresses too

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.device = self._held[0].device  # a loaded cache may have been sent elsewhere
        if self.device.type != "cuda":
            raise ValueError(f"tda_amd runs on the GPU only (HIP); got a cache on {self.device}")

    # -------------------------------------------------------------- calls
    def _cache(self) -> _sda_abi.SdaKv4:
        c = _sda_abi.SdaKv4()
        c.batch, c.kv_heads, c.capacity = self.batch, self.kv_heads, self.capacity
        c.head_dim, c.v_head_dim = self.head_dim, self.v_head_dim
        c.k1, c.k2, c.v = (t.data_ptr() for t in self._held)
        return c

    def _template(self, key, build):
        """The argument block of a call but for the call's own pointers, cached by its configuration (this
        cache's buffers are part of it)."""
        n = self.lengths
        if not isinstance(n, torch.Tensor) or n.shape != (self.batch,) or n.dtype != torch.int32 or n.device != self.device \
                or not n.is_contiguous():
            raise ValueError(f"lengths must be a contiguous int32 tensor of shape ({self.batch},) on {self.device}")
        got = self._templates.get(key)
        if got is None:
            if len(self._templates) > 64:
                self._templates.clear()
            block = build()
            got = self._templates[key] = bytes(block), getattr(block, "workspace_bytes", 0)
        buf = bytearray(got[0])
        _PUT(buf, _LENGTHS, n.data_ptr())
        return buf, got[1]

    def _signature(self, *tensors):
        """What a call's plan goes by (the lengths' form among it), or None."""
        for t in (self.lengths, *tensors):
            if t is not None and type(t) not in _TENSORS:
                return None
        if self.lengths is None:
            return None
        return _sig(self.lengths), *[None if t is None else _sig(t) for t in tensors]

    def _planned(self, key, rows):
        """(argument block, ...) that _plan kept for calls of this signature; None where there is none, or
        where an address does not suit the kernels."""
        got = self._plans.get(key)
        if got is None:
            return None
        for t in rows:
            if t.data_ptr() % 16:
                return None
        buf = bytearray(got[0])
        _PUT(buf, _LENGTHS, self.lengths.data_ptr())
        return buf, *got[1:]

    def _plan(self, key, *plan):
        if key is not None:
            if len(self._plans) > 64:
                self._plans.clear()
            self._plans[key] = plan

    def _check(self, tensors, names, shapes):
        _check_rows(tensors, names)
        for t, n, s in zip(tensors, names, shapes):
            if t.shape != s:
                raise ValueError(f"{n} must have shape {tuple(s)}, got {tuple(t.shape)}")
        if tensors[0].device != self.device:
            raise ValueError(f"device mismatch: the cache is on {self.device}, {names[0]} on {tensors[0].device}")
        if tensors[0].dtype not in _CODE:
            raise ValueError(f"unsupported dtype {tensors[0].dtype}")

    def append(self, k1, k2, v, counts=None, start=None):
        """Add the rows of new positions: k1, k2 (batch, kv_heads, n, head_dim), v (..., n, v_head_dim),
        float32, bfloat16 or float16, n <= capacity.

        Row i of sequence b goes to position lengths[b] + i, or start[b] + i where start (int32/int64,
        (batch,)) is given, for i < counts[b] (all n by default; rows past it are padding and are not
        read); lengths[b] becomes the position behind the last one.  Positions outside 0 .. capacity - 1
        are dropped, and lengths stops at the capacity: a caller that must not lose rows keeps count.  start and
        counts may be `lengths` itself, but no other tensor that overlaps it."""
        key = self._signature(k1, k2, v, start, counts)
        plan = self._planned(key, (k1, k2, v)) if key is not None else None
        if plan is not None:
            self._append(plan[0], k1, k2, v, start, counts)
            return
        n = k1.shape[2] if isinstance(k1, torch.Tensor) and k1.dim() == 4 else 0
        b, hk = self.batch, self.kv_heads
        given = k1, k2, v, start, counts
        self._check((k1, k2, v), ("k1", "k2", "v"),
                    ((b, hk, n, self.head_dim), (b, hk, n, self.head_dim), (b, hk, n, self.v_head_dim)))
        if n > self.capacity:
            raise ValueError(f"{n} rows do not fit a cache of {self.capacity}")
        counts = None if counts is None else _ints(counts, b, self.device, "counts")
        start = None if start is None else _ints(start, b, self.device, "start")
        if n == 0:
            if start is not None:
                self.lengths.copy_(start.clamp(0, self.capacity))
            return
        self._wide |= k1.dtype != torch.float16
        rows = [_usable(t) for t in (k1, k2, v)]

        def build():
            a = _sda_abi.SdaKv4AppendArgs()
            a.abi_version, a.dtype, a.cache, a.rows = _sda_abi.ABI_VERSION, _CODE[rows[0].dtype], self._cache(), n
            for name, t in zip(("k1", "k2", "v"), rows):
                getattr(a, name).stride[:] = t.stride()
            return a

        buf, _ = self._template(("append", n, rows[0].dtype, tuple(t.stride() for t in rows)), build)
        if all(a is b for a, b in zip((*rows, start, counts), given)):
            self._plan(key, bytes(buf))
        self._append(buf, *rows, start, counts)

    def _append(self, buf, *tensors):
        for name, t in zip(("k1", "k2", "v", "start", "counts"), tensors):
            if t is not None:
                _PUT(buf, _APPEND_OFF[name], t.data_ptr())
        _launch(_sda_abi.load().sda_kv4_append, _sda_abi.SdaKv4AppendArgs, buf, self.device, "sda_kv4_append")

    def read(self, rows: int | None = None, dtype=torch.bfloat16):
        """The first `rows` (default: capacity) positions as tensors k1, k2, v of a dtype; positions a
        sequence does not hold are zero.  In float16 values past +-65504 (held from rows of a wider type, or a
        step beyond float16 rows next to that) read as +-65504."""
        n = self.capacity if rows is None else int(rows)
        if not 1 <= n <= self.capacity:
            raise ValueError(f"rows must be 1 to {self.capacity}, got {n}")
        if dtype not in _CODE:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        res = tuple(torch.empty((self.batch, self.kv_heads, n, w), dtype=dtype, device=self.device)
                    for w in (self.head_dim, self.head_dim, self.v_head_dim))

        def build():
            a = _sda_abi.SdaKv4ReadArgs()
            a.abi_version, a.dtype, a.cache, a.rows = _sda_abi.ABI_VERSION, _CODE[dtype], self._cache(), n
            for name, t in zip(("k1", "k2", "v"), res):
                getattr(a, name).stride[:] = t.stride()
            return a

        buf, _ = self._template(("read", n, dtype), build)
        for name, t in zip(("k1", "k2", "v"), res):
            _PUT(buf, _READ_OFF[name], t.data_ptr())
        _launch(_sda_abi.load().sda_kv4_read, _sda_abi.SdaKv4ReadArgs, buf, self.device, "sda_kv4_read")
        return res

    def attend(self, q1, q2, lambda_param, scale=None):
        """Softmax differential attention of q1, q2 (batch, heads, n, head_dim), the last n positions of each
        sequence, over the cache: row i of sequence b sees the keys up to lengths[b] - n + i (a row before
        the sequence's first position is zero).  Returns (batch, heads, n, v_head_dim); no gradient.
        (A group of values that is not finite reaches the rows that see it, and may reach other rows of
        the same call that stand before it.)

        The rows of a decoding step or of a short chunk are computed from the codes; those of a long
        one from the rows that read() gives in q1's dtype, unless that is float16 and the cache took rows of
        another type, whose range float16 may not hold."""
        key = self._signature(q1, q2, lambda_param) if scale is None or type(scale) is float else None
        if key is not None:
            key = *key, scale
            plan = self._planned(key, (q1, q2))
            if plan is not None:
                buf, size, shape, strides = plan
                return self._attend(buf, size, q1, q2, lambda_param,
                                    torch.empty_strided(shape, strides, dtype=q1.dtype, device=self.device))
        given = q1, q2, lambda_param
        b, hk = self.batch, self.kv_heads
        if isinstance(q1, torch.Tensor) and q1.dim() == 4:
            h, n = q1.shape[1], q1.shape[2]
        else:
            h, n = hk, 0
        self._check((q1, q2), ("q1", "q2"), ((b, h, n, self.head_dim),) * 2)
        _check_heads(h, hk)
        s = _scale(scale, self.head_dim)
        lam = _lambda(lambda_param, b, h, n, self.device)
        if n == 0:
            return torch.zeros((b, h, 0, self.v_head_dim), dtype=q1.dtype, device=self.device)
        narrow = q1.dtype == torch.float16 and self._wide
        if not narrow and not _from_codes(b, hk, h // hk * n, q1.dtype):
            with torch.no_grad():
                rows = self.read(dtype=q1.dtype)  # checks lengths
                lens = self.lengths.clamp(0, self.capacity)
                return differential_attention(q1, q2, *rows, lam, s, q_offset=lens - n, kv_lens=lens)
        q1, q2 = _usable(q1), _usable(q2)
        out = _new_rows(q1, self.v_head_dim)
        ls = _lambda_strides(lam)

        def build():
            a = _sda_abi.SdaKv4AttendArgs()
            a.abi_version, a.dtype, a.cache = _sda_abi.ABI_VERSION, _CODE[q1.dtype], self._cache()
            a.heads, a.seq_len, a.scale = h, n, s
            for name, t in zip(("q1", "q2", "out"), (q1, q2, out)):
                getattr(a, name).stride[:] = t.stride()
            a.lambda_stride[:] = ls
            a.lambda_dtype = _CODE[lam.dtype]
            a.workspace_bytes = _sda_abi.load().sda_kv4_attend_workspace_bytes(ctypes.byref(a))
            return a

        buf, size = self._template(("attend", h, n, s, q1.dtype, lam.dtype, ls, q1.stride(), q2.stride()), build)
        if all(a is b for a, b in zip((q1, q2, lam), given)):
            self._plan(key, bytes(buf), size, out.shape, out.stride())
        return self._attend(buf, size, q1, q2, lam, out)

    def _attend(self, buf, size, q1, q2, lam, out):
        ws = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        for name, t in zip(("q1", "q2", "out", "lambda_param", "workspace"), (q1, q2, out, lam, ws)):
            if t is not None:
                _PUT(buf, _ATTEND_OFF[name], t.data_ptr())
        _launch(_sda_abi.load().sda_kv4_attend, _sda_abi.SdaKv4AttendArgs, buf, self.device, "sda_kv4_attend")
        return out
