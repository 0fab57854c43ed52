"""C ABI of the softmax differential attention operators (include/sda.h): the library exports what the
header declares, the ctypes mirror has its layout, and every argument that lies in host memory is checked
before a launch.  No GPU needed."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from tda_amd import _abi, _sda_abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sda.h")
FAKE = 0x10000  # aligned, never read: the checks are host code


def lib():
    if not os.path.exists(_abi.lib_path()):
        pytest.skip("libtda_hip.so not built (python -m tda_amd.build)")
    return _sda_abi.load()


def test_header_and_library_agree():
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(sda_\w+)\s*\(", open(HEADER).read(), re.M))
    assert names == set(_sda_abi.SIGNATURES)
    so = lib()
    assert all(hasattr(so, n) for n in names) and so.sda_abi_version() == _sda_abi.ABI_VERSION


def test_struct_layouts(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc missing")
    structs = {"sda_fwd_args": _sda_abi.SdaFwdArgs, "sda_bwd_args": _sda_abi.SdaBwdArgs, "sda_rotary_args": _sda_abi.SdaRotaryArgs,
               "sda_kv4": _sda_abi.SdaKv4, "sda_kv4_append_args": _sda_abi.SdaKv4AppendArgs,
               "sda_kv4_read_args": _sda_abi.SdaKv4ReadArgs, "sda_kv4_attend_args": _sda_abi.SdaKv4AttendArgs}
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run([gcc, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {tuple(ln.split()[:2]): int(ln.split()[2]) for ln in out if ln}
    for c, py in structs.items():
        assert got[c, "size"] == ctypes.sizeof(py), c
        assert all(got[c, f] == getattr(py, f).offset for f, _ in py._fields_), c


def _rows(shape):
    t = _abi.TdaTensor()
    b, h, n, d = shape
    t.data, t.stride[:] = FAKE, (h * n * d, n * d, d, 1)
    return t


def _common(a, b=2, h=4, hk=2, n=100, nk=130, d=64, dv=128):
    a.abi_version, a.dtype, a.causal, a.scale = _sda_abi.ABI_VERSION, _abi.DTYPE_BF16, 1, 0.125
    a.batch, a.heads, a.kv_heads, a.seq_len, a.seq_len_kv, a.head_dim, a.v_head_dim = b, h, hk, n, nk, d, dv
    a.q1 = a.q2 = _rows((b, h, n, d))
    a.k1 = a.k2 = _rows((b, hk, nk, d))
    a.v, a.out = _rows((b, hk, nk, dv)), _rows((b, h, n, dv))
    a.lambda_param, a.lambda_dtype, a.q_offset = FAKE, _abi.DTYPE_F32, 30
    return a


def fwd(**kw):
    a = _common(_sda_abi.SdaFwdArgs(), **kw)
    a.workspace, a.workspace_bytes = FAKE, lib().sda_fwd_workspace_bytes(ctypes.byref(a))
    return a


def bwd(**kw):
    a = _common(_sda_abi.SdaBwdArgs(), **kw)
    a.out2 = _rows((a.batch, a.heads, a.seq_len, a.v_head_dim))
    for n, like in (("out_low", "out"), ("dout", "out"), ("dq1", "q1"), ("dq2", "q2"), ("dk1", "k1"), ("dk2", "k2"), ("dv", "v")):
        setattr(a, n, getattr(a, like))
    a.lse = a.workspace = FAKE
    a.workspace_bytes = lib().sda_bwd_workspace_bytes(ctypes.byref(a))
    return a


BAD_ROWS = [
    (lambda a: setattr(a, "abi_version", 7), _abi.ERR_ABI),
    (lambda a: setattr(a, "dtype", 3), _abi.ERR_DTYPE),
    (lambda a: setattr(a, "causal", 2), _abi.ERR_CAUSAL),
    (lambda a: setattr(a, "scale", 0.0), _sda_abi.ERR_SCALE),
    (lambda a: setattr(a, "scale", float("nan")), _sda_abi.ERR_SCALE),
    (lambda a: setattr(a, "scale", float("inf")), _sda_abi.ERR_SCALE),
    (lambda a: setattr(a, "batch", 0), _abi.ERR_SHAPE),
    (lambda a: setattr(a, "seq_len", 0), _abi.ERR_SHAPE),
    (lambda a: setattr(a, "seq_len_kv", -1), _abi.ERR_SHAPE),
    (lambda a: setattr(a, "heads", 5), _sda_abi.ERR_HEADS),
    (lambda a: setattr(a, "head_dim", 32), _abi.ERR_HEAD_DIM),
    (lambda a: setattr(a, "v_head_dim", 256), _abi.ERR_HEAD_DIM),
    (lambda a: setattr(a, "seq_len_kv", 1 << 30), _abi.ERR_OFFSET),
    (lambda a: setattr(a, "q_offset", 1 << 30), _abi.ERR_OFFSET),
    (lambda a: setattr(a, "batch", 1 << 29), _abi.ERR_SHAPE),
    (lambda a: setattr(a, "lambda_param", None), _abi.ERR_NULL_POINTER),
    (lambda a: setattr(a, "lambda_param", FAKE + 2), _abi.ERR_LAYOUT),
    (lambda a: setattr(a, "lambda_dtype", 3), _abi.ERR_DTYPE),
    (lambda a: a.lambda_stride.__setitem__(1, -1), _abi.ERR_LAYOUT),
    (lambda a: setattr(a.q2, "data", None), _abi.ERR_NULL_POINTER),
    (lambda a: setattr(a.v, "data", FAKE + 8), _abi.ERR_LAYOUT),
    (lambda a: a.k1.stride.__setitem__(3, 2), _abi.ERR_LAYOUT),
    (lambda a: a.k1.stride.__setitem__(2, 65), _abi.ERR_LAYOUT),
    (lambda a: a.k1.stride.__setitem__(2, (1 << 24) + 8), _abi.ERR_LAYOUT),
    (lambda a: a.out.stride.__setitem__(0, -64), _abi.ERR_LAYOUT),
]


@pytest.mark.parametrize("mutate, code", BAD_ROWS)
def test_attention_refuses(mutate, code):
    so = lib()
    for a, check, call in ((fwd(), so.sda_validate_fwd, so.sda_fwd), (bwd(), so.sda_validate_bwd, so.sda_bwd)):
        assert check(ctypes.byref(a)) == _abi.OK
        mutate(a)
        assert check(ctypes.byref(a)) == code and call(ctypes.byref(a), None) == code
    assert so.sda_validate_fwd(None) == so.sda_validate_bwd(None) == _abi.ERR_NULL_POINTER


def test_attention_workspaces():
    so = lib()
    assert fwd(n=2000, nk=2000).workspace_bytes == 0  # many rows: no key split
    a = fwd(n=1, nk=5000)
    # 4 items of 2 rows, keys in parts of 128: 40 parts
    assert a.workspace_bytes == 4 * 40 * (64 + 32 * 128) * 4
    assert so.sda_validate_fwd(ctypes.byref(a)) == _abi.OK
    for at, size in ((None, a.workspace_bytes), (FAKE, a.workspace_bytes - 4), (FAKE + 4, a.workspace_bytes)):
        a.workspace, a.workspace_bytes = at, size
        assert so.sda_validate_fwd(ctypes.byref(a)) == _abi.ERR_WORKSPACE
        a.workspace_bytes = so.sda_fwd_workspace_bytes(ctypes.byref(a))
    a.lse = FAKE  # a training forward keeps to the tile kernels
    assert so.sda_fwd_workspace_bytes(ctypes.byref(a)) == 0
    b = bwd()
    assert b.workspace_bytes >= 3 * 2 * 4 * 100 * 4
    b.workspace_bytes -= 4
    assert so.sda_validate_bwd(ctypes.byref(b)) == _abi.ERR_WORKSPACE
    b = bwd()
    b.lse = None
    assert so.sda_validate_bwd(ctypes.byref(b)) == _abi.ERR_NULL_POINTER
    for name in ("out2", "out_low"):  # what the forward keeps; f32 needs no low part
        b = bwd()
        getattr(b, name).data = None
        assert so.sda_validate_bwd(ctypes.byref(b)) == _abi.ERR_NULL_POINTER
        b.dtype = _abi.DTYPE_F32
        assert so.sda_validate_bwd(ctypes.byref(b)) == (_abi.OK if name == "out_low" else _abi.ERR_NULL_POINTER)
    assert so.sda_fwd_workspace_bytes(None) == so.sda_bwd_workspace_bytes(None) == so.sda_kv4_attend_workspace_bytes(None) == 0


def rotary():
    a = _sda_abi.SdaRotaryArgs()
    a.abi_version, a.dtype, a.batch, a.seq_len, a.head_dim, a.rot = _sda_abi.ABI_VERSION, _sda_abi.DTYPE_F16, 2, 5, 64, 48
    a.axes, a.count, a.position_dtype = 3, 2, 8
    a.sections[:] = (8, 8, 8, 0)
    for i in range(2):
        a.heads[i], a.x[i], a.y[i] = 3, _rows((2, 3, 5, 64)), _rows((2, 3, 5, 64))
    a.positions = a.inv_freq = FAKE
    a.position_stride[:] = (10, 5, 1)
    return a


@pytest.mark.parametrize("mutate, code", [
    (lambda a: setattr(a, "abi_version", 0), _abi.ERR_ABI), (lambda a: setattr(a, "dtype", 3), _abi.ERR_DTYPE),
    (lambda a: setattr(a, "position_dtype", 2), _abi.ERR_DTYPE), (lambda a: setattr(a, "seq_len", 0), _abi.ERR_SHAPE),
    (lambda a: setattr(a, "head_dim", 9000), _abi.ERR_SHAPE), (lambda a: setattr(a, "axes", 0), _sda_abi.ERR_AXES),
    (lambda a: setattr(a, "axes", 5), _sda_abi.ERR_AXES), (lambda a: setattr(a, "count", 5), _sda_abi.ERR_AXES),
    (lambda a: setattr(a, "rot", 47), _sda_abi.ERR_AXES), (lambda a: setattr(a, "rot", 66), _sda_abi.ERR_AXES),
    (lambda a: a.sections.__setitem__(0, 7), _sda_abi.ERR_AXES), (lambda a: a.sections.__setitem__(1, -8), _sda_abi.ERR_AXES),
    (lambda a: setattr(a, "positions", None), _abi.ERR_NULL_POINTER), (lambda a: setattr(a, "positions", FAKE + 4), _abi.ERR_LAYOUT),
    (lambda a: setattr(a, "inv_freq", None), _abi.ERR_NULL_POINTER), (lambda a: a.heads.__setitem__(1, 0), _abi.ERR_SHAPE),
    (lambda a: setattr(a.x[1], "data", None), _abi.ERR_NULL_POINTER), (lambda a: setattr(a.y[0], "data", FAKE + 1), _abi.ERR_LAYOUT),
    (lambda a: a.x[0].stride.__setitem__(3, 2), _abi.ERR_LAYOUT), (lambda a: a.position_stride.__setitem__(0, -1), _abi.ERR_LAYOUT)])
def test_rotary_refuses(mutate, code):
    so, a = lib(), rotary()
    assert so.sda_validate_rotary(ctypes.byref(a)) == _abi.OK
    mutate(a)
    assert so.sda_validate_rotary(ctypes.byref(a)) == code and so.sda_rotary(ctypes.byref(a), None) == code
    assert so.sda_validate_rotary(None) == _abi.ERR_NULL_POINTER


def _cache(a):
    a.abi_version, a.dtype = _sda_abi.ABI_VERSION, _abi.DTYPE_BF16
    c = a.cache
    c.batch, c.kv_heads, c.capacity, c.head_dim, c.v_head_dim = 2, 2, 500, 64, 128
    c.k1 = c.k2 = c.v = c.lengths = FAKE
    return a


def kv4(cls):
    a = _cache(cls())
    if cls is _sda_abi.SdaKv4AttendArgs:
        a.heads, a.seq_len, a.scale = 4, 1, 0.125
        a.q1 = a.q2 = _rows((2, 4, 1, 64))
        a.out = _rows((2, 4, 1, 128))
        a.lambda_param = a.workspace = FAKE
        a.workspace_bytes = lib().sda_kv4_attend_workspace_bytes(ctypes.byref(a))
    else:
        a.rows = 3
        a.k1 = a.k2 = _rows((2, 2, 3, 64))
        a.v = _rows((2, 2, 3, 128))
    return a


KINDS = {"append": _sda_abi.SdaKv4AppendArgs, "read": _sda_abi.SdaKv4ReadArgs, "attend": _sda_abi.SdaKv4AttendArgs}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mutate, code", [
    (lambda a: setattr(a, "abi_version", 0), _abi.ERR_ABI), (lambda a: setattr(a, "dtype", 3), _abi.ERR_DTYPE),
    (lambda a: setattr(a.cache, "batch", 0), _abi.ERR_SHAPE), (lambda a: setattr(a.cache, "head_dim", 96), _abi.ERR_HEAD_DIM),
    (lambda a: setattr(a.cache, "capacity", (1 << 24) + 1), _sda_abi.ERR_CACHE),
    (lambda a: setattr(a.cache, "k2", None), _abi.ERR_NULL_POINTER), (lambda a: setattr(a.cache, "lengths", None), _abi.ERR_NULL_POINTER),
    (lambda a: setattr(a.cache, "v", FAKE + 8), _abi.ERR_LAYOUT), (lambda a: setattr(a.cache, "lengths", FAKE + 2), _abi.ERR_LAYOUT)])
def test_cache_refuses(kind, mutate, code):
    so, a = lib(), kv4(KINDS[kind])
    check, call = getattr(so, f"sda_validate_kv4_{kind}"), getattr(so, f"sda_kv4_{kind}")
    assert check(ctypes.byref(a)) == _abi.OK
    mutate(a)
    assert check(ctypes.byref(a)) == code and call(ctypes.byref(a), None) == code
    assert check(None) == _abi.ERR_NULL_POINTER


@pytest.mark.parametrize("kind, mutate, code", [
    ("append", lambda a: setattr(a, "rows", 501), _sda_abi.ERR_CACHE), ("append", lambda a: setattr(a, "rows", 0), _sda_abi.ERR_CACHE),
    ("append", lambda a: setattr(a.v, "data", None), _abi.ERR_NULL_POINTER), ("append", lambda a: setattr(a.k1, "data", FAKE + 2), _abi.ERR_LAYOUT),
    ("read", lambda a: setattr(a, "rows", 501), _sda_abi.ERR_CACHE), ("read", lambda a: a.k2.stride.__setitem__(3, 2), _abi.ERR_LAYOUT),
    ("attend", lambda a: setattr(a, "heads", 3), _sda_abi.ERR_HEADS), ("attend", lambda a: setattr(a, "seq_len", 0), _abi.ERR_SHAPE),
    ("attend", lambda a: setattr(a, "scale", -1.0), _sda_abi.ERR_SCALE), ("attend", lambda a: setattr(a, "lambda_param", None), _abi.ERR_NULL_POINTER),
    ("attend", lambda a: setattr(a, "workspace", None), _abi.ERR_WORKSPACE),
    ("attend", lambda a: setattr(a, "workspace_bytes", a.workspace_bytes - 1), _abi.ERR_WORKSPACE),
    ("attend", lambda a: setattr(a.out, "data", None), _abi.ERR_NULL_POINTER)])
def test_cache_refuses_its_own(kind, mutate, code):
    so, a = lib(), kv4(KINDS[kind])
    mutate(a)
    assert getattr(so, f"sda_validate_kv4_{kind}")(ctypes.byref(a)) == code
    assert getattr(so, f"sda_kv4_{kind}")(ctypes.byref(a), None) == code


def test_cache_sizes_and_error_strings():
    so = lib()
    assert so.sda_kv4_bytes(2, 3, 10, 128) == 2 * 3 * 12 * (64 + 8)  # rows in fours
    assert so.sda_kv4_bytes(2, 3, 10, 96) == so.sda_kv4_bytes(0, 3, 10, 64) == 0
    texts = [so.sda_error_string(c).decode() for c in (*range(-13, 0), *range(-23, -19), -100)]
    assert all(texts) and len(set(texts[-5:])) == 5


def test_append_refuses_arrays_that_overlap_the_lengths():
    """The kernel writes the lengths while it reads start and counts."""
    so = lib()
    for name in ("start", "counts"):
        for apart, code in ((0, _abi.OK), (4, _sda_abi.ERR_CACHE), (-4, _sda_abi.ERR_CACHE), (8, _abi.OK), (-8, _abi.OK)):
            a = kv4(_sda_abi.SdaKv4AppendArgs)
            setattr(a, name, FAKE + apart)
            assert so.sda_validate_kv4_append(ctypes.byref(a)) == code, (name, apart)


@pytest.mark.parametrize("name, width", [("q1", 64), ("q2", 64), ("dout", 128)])
@pytest.mark.parametrize("n, code", [(1, _abi.ERR_LAYOUT), (33, _abi.ERR_LAYOUT), (100, _abi.ERR_LAYOUT), (32, _abi.OK), (96, _abi.OK)])
def test_backward_refuses_query_rows_that_overlap(name, width, n, code):
    """Its last tile of 32 rows reads past them, where overlapping rows are not zeros."""
    so = lib()
    for step in (0, 8, width - 8, width):
        a = bwd(n=n)
        t = _rows((2, 4, n, width))
        t.stride[2] = step
        setattr(a, name, t)
        assert so.sda_validate_bwd(ctypes.byref(a)) == (_abi.OK if step == width else code)
