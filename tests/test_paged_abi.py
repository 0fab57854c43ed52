"""C ABIs of the paged cache (include/spa.h) and the layer norm (include/sln.h): the library exports what the headers
declare, the ctypes mirrors have their layouts, and every argument that lies in host memory is checked before a launch.
No GPU needed."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from tda_amd import _abi, _sda_abi, _sln_abi, _spa_abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x10000  # aligned, never read: the checks are host code
ABIS = {"spa": _spa_abi, "sln": _sln_abi}


def lib():
    if not os.path.exists(_abi.lib_path()):
        pytest.skip("libtda_hip.so not built (python -m tda_amd.build)")
    _spa_abi.load()
    return _sln_abi.load()


@pytest.mark.parametrize("name", ABIS)
def test_header_and_library_agree(name):
    text = open(os.path.join(ROOT, "include", f"{name}.h")).read()
    names = set(re.findall(rf"^\s*(?:const\s+)?\w+\s*\*?\s*({name}_\w+)\s*\(", text, re.M))
    assert names == set(ABIS[name].SIGNATURES)
    so = lib()
    assert all(hasattr(so, n) for n in names) and getattr(so, f"{name}_abi_version")() == ABIS[name].ABI_VERSION


def test_struct_layouts(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc missing")
    structs = {"spa_cache": _spa_abi.SpaCache, "spa_rows": _spa_abi.SpaRows, "spa_append_args": _spa_abi.SpaAppendArgs,
               "spa_attend_args": _spa_abi.SpaAttendArgs, "sln_fwd_args": _sln_abi.SlnFwdArgs, "sln_bwd_args": _sln_abi.SlnBwdArgs}
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", *[f'#include "{ROOT}/include/{n}.h"' for n in ABIS], "int main(void){"]
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


def _rows(b, h, n, d):
    t = _abi.TdaTensor()
    t.data, t.stride[:] = FAKE, (h * n * d, n * d, d, 1)
    return t


def _cache(a, pages=10, hk=2, page=16, d=64, dv=128):
    c = a.cache
    c.pages, c.kv_heads, c.page_size, c.head_dim, c.v_head_dim = pages, hk, page, d, dv
    c.k1 = c.k2 = c.v = FAKE


def _at(a, s=3, n=5, table_len=100):
    a.at.sequences, a.at.rows, a.at.table, a.at.table_stride, a.at.table_len, a.at.lengths = s, n, FAKE, table_len, table_len, FAKE


def append():
    a = _spa_abi.SpaAppendArgs()
    a.abi_version, a.dtype = _spa_abi.ABI_VERSION, _abi.DTYPE_BF16
    _cache(a)
    _at(a)
    a.k1 = a.k2 = _rows(3, 2, 5, 64)
    a.v = _rows(3, 2, 5, 128)
    a.heads, a.rot, a.axes, a.inv_freq = 4, 48, 2, FAKE
    a.q1 = a.q2 = a.q1_out = a.q2_out = _rows(3, 4, 5, 64)
    a.sections[:2] = 14, 10
    a.positions, a.position_dtype, a.position_stride[:] = FAKE, 8, (15, 5, 1)
    return a


def attend(**kw):
    a = _spa_abi.SpaAttendArgs()
    a.abi_version, a.dtype, a.scale = _spa_abi.ABI_VERSION, _abi.DTYPE_BF16, 0.125
    _cache(a)
    _at(a, **kw)
    a.heads, a.lambda_param, a.lambda_dtype = 4, FAKE, _abi.DTYPE_F32
    s, n = a.at.sequences, a.at.rows
    a.q1 = a.q2 = _rows(s, 4, n, 64)
    a.out = _rows(s, 4, n, 128)
    a.workspace, a.workspace_bytes = FAKE, lib().spa_attend_workspace_bytes(ctypes.byref(a))
    return a


def put(path, value):
    def change(a):
        *way, last = path.split(".")
        for w in way:
            a = getattr(a, w)
        if "[" in last:
            name, i = last[:-1].split("[")
            getattr(a, name)[int(i)] = value
        else:
            setattr(a, last, value)
    return change


BOTH = [("abi_version", 9, _abi.ERR_ABI), ("dtype", 3, _abi.ERR_DTYPE), ("cache.pages", 0, _spa_abi.ERR_PAGES), ("cache.pages", 1 << 31, _spa_abi.ERR_PAGES),
        ("cache.page_size", 8, _spa_abi.ERR_PAGES), ("cache.page_size", 48, _spa_abi.ERR_PAGES), ("cache.page_size", 512, _spa_abi.ERR_PAGES),
        ("cache.page_size", -16, _spa_abi.ERR_PAGES), ("cache.kv_heads", 0, _abi.ERR_SHAPE), ("cache.head_dim", 96, _abi.ERR_HEAD_DIM),
        ("cache.v_head_dim", 256, _abi.ERR_HEAD_DIM), ("cache.k1", None, _abi.ERR_NULL_POINTER), ("cache.v", FAKE + 8, _abi.ERR_LAYOUT),
        ("at.sequences", 0, _abi.ERR_SHAPE), ("at.rows", 0, _abi.ERR_SHAPE), ("at.rows", 1 << 40, _abi.ERR_SHAPE), ("at.table", None, _abi.ERR_NULL_POINTER),
        ("at.lengths", None, _abi.ERR_NULL_POINTER), ("at.table_len", 0, _spa_abi.ERR_PAGES), ("at.table_len", 1 << 28, _spa_abi.ERR_PAGES),
        ("at.table_stride", -1, _spa_abi.ERR_PAGES), ("at.table", FAKE + 2, _abi.ERR_LAYOUT), ("at.lengths", FAKE + 1, _abi.ERR_LAYOUT),
        ("at.counts", FAKE + 2, _abi.ERR_LAYOUT), ("q1.data", None, _abi.ERR_NULL_POINTER), ("q2.stride[3]", 2, _abi.ERR_LAYOUT),
        ("q1.stride[2]", 4, _abi.ERR_LAYOUT), ("q1.stride[0]", -64, _abi.ERR_LAYOUT), ("q2.stride[2]", 1 << 25, _abi.ERR_LAYOUT)]


@pytest.mark.parametrize("path, value, code", BOTH + [
    ("heads", -1, _abi.ERR_SHAPE), ("q1_out.data", FAKE + 4, _abi.ERR_LAYOUT), ("k2.data", None, _abi.ERR_NULL_POINTER), ("v.stride[1]", 3, _abi.ERR_LAYOUT),
    ("rot", 47, _sda_abi.ERR_AXES), ("rot", 66, _sda_abi.ERR_AXES), ("rot", -2, _sda_abi.ERR_AXES), ("axes", 0, _sda_abi.ERR_AXES),
    ("axes", 5, _sda_abi.ERR_AXES), ("sections[0]", 15, _sda_abi.ERR_AXES), ("sections[0]", -14, _sda_abi.ERR_AXES), ("inv_freq", None, _abi.ERR_NULL_POINTER),
    ("inv_freq", FAKE + 2, _abi.ERR_LAYOUT), ("position_dtype", 2, _abi.ERR_DTYPE), ("positions", FAKE + 4, _abi.ERR_LAYOUT),
    ("position_stride[1]", -1, _abi.ERR_LAYOUT)])
def test_append_refuses(path, value, code):
    a = append()
    assert lib().spa_validate_append(ctypes.byref(a)) == _abi.OK
    put(path, value)(a)
    assert lib().spa_validate_append(ctypes.byref(a)) == lib().spa_append(ctypes.byref(a), None) == code


@pytest.mark.parametrize("path, value, code", BOTH + [
    ("heads", 0, _abi.ERR_SHAPE), ("heads", 3, _sda_abi.ERR_HEADS), ("most", -1, _abi.ERR_SHAPE), ("scale", 0.0, _sda_abi.ERR_SCALE),
    ("scale", float("nan"), _sda_abi.ERR_SCALE), ("lambda_param", None, _abi.ERR_NULL_POINTER), ("lambda_param", FAKE + 2, _abi.ERR_LAYOUT),
    ("lambda_dtype", 7, _abi.ERR_DTYPE), ("lambda_stride[0]", -1, _abi.ERR_LAYOUT), ("out.data", None, _abi.ERR_NULL_POINTER),
    ("workspace", None, _abi.ERR_WORKSPACE), ("workspace", FAKE + 8, _abi.ERR_WORKSPACE), ("workspace_bytes", 100, _abi.ERR_WORKSPACE)])
def test_attend_refuses(path, value, code):
    a = attend()
    assert a.workspace_bytes and lib().spa_validate_attend(ctypes.byref(a)) == _abi.OK
    put(path, value)(a)
    assert lib().spa_validate_attend(ctypes.byref(a)) == lib().spa_attend(ctypes.byref(a), None) == code


def test_starts_and_counts_exclude_each_other_and_null_is_refused():
    for a, fn in ((append(), "append"), (attend(), "attend")):
        a.at.starts = a.at.counts = FAKE
        assert getattr(lib(), f"spa_validate_{fn}")(ctypes.byref(a)) == _spa_abi.ERR_ROWS
        assert getattr(lib(), f"spa_validate_{fn}")(None) == getattr(lib(), f"spa_{fn}")(None, None) == _abi.ERR_NULL_POINTER
    a = append()  # what is not used is not checked
    a.heads, a.rot, a.axes, a.inv_freq, a.positions = 0, 0, 0, None, None
    a.q1.data = a.q2.data = a.q1_out.data = None
    assert lib().spa_validate_append(ctypes.byref(a)) == _abi.OK


def test_attend_workspaces():
    """None where the tiles fill the chip; two places for sums for each workgroup where they do not, of either form of rows."""
    few, many = (64 + 2 * 16 * 128) * 4, (4 * 128 + 2 * 128 * 128) * 4
    assert attend(s=3, n=5).workspace_bytes == 512 * few
    assert attend(s=3, n=100).workspace_bytes == 512 * many
    a = attend(s=3, n=5)
    a.at.table_len = 4  # 256 positions
    assert lib().spa_attend_workspace_bytes(ctypes.byref(a)) == 0
    assert attend(s=30000, n=5).workspace_bytes == attend(s=300, n=100).workspace_bytes == 0
    a = attend(s=3, n=100)
    a.at.counts = FAKE
    assert lib().spa_attend_workspace_bytes(ctypes.byref(a)) == 512 * many
    a.most = 8
    assert lib().spa_attend_workspace_bytes(ctypes.byref(a)) == 512 * few
    a.heads = 3
    assert lib().spa_attend_workspace_bytes(ctypes.byref(a)) == lib().spa_attend_workspace_bytes(None) == 0


# ------------------------------------------------------------------ layer norm
def fwd():
    a = _sln_abi.SlnFwdArgs()
    a.abi_version, a.dtype, a.weight_dtype, a.eps, a.center = _sln_abi.ABI_VERSION, _abi.DTYPE_BF16, _abi.DTYPE_F32, 1e-5, 1
    a.batch, a.heads, a.rows, a.width = 2, 3, 700, 100
    a.x = a.y = _rows(2, 3, 700, 100)
    a.weight = a.bias = a.stats = FAKE
    return a


def bwd():
    a = _sln_abi.SlnBwdArgs()
    a.abi_version, a.dtype, a.weight_dtype = _sln_abi.ABI_VERSION, _abi.DTYPE_BF16, _abi.DTYPE_F32
    a.batch, a.heads, a.rows, a.width = 2, 3, 700, 100
    a.x = a.dy = a.dx = _rows(2, 3, 700, 100)
    a.weight = a.stats = a.dweight = a.dbias = FAKE
    a.workspace, a.workspace_bytes = FAKE, lib().sln_bwd_workspace_bytes(ctypes.byref(a))
    return a


NORM = [("abi_version", 0, _abi.ERR_ABI), ("dtype", 5, _abi.ERR_DTYPE), ("weight_dtype", _sda_abi.DTYPE_F16, _abi.ERR_DTYPE), ("batch", 0, _abi.ERR_SHAPE),
        ("rows", -1, _abi.ERR_SHAPE), ("rows", 1 << 30, _abi.ERR_SHAPE), ("width", 0, _sln_abi.ERR_WIDTH), ("width", 16385, _sln_abi.ERR_WIDTH),
        ("x.data", None, _abi.ERR_NULL_POINTER), ("x.data", FAKE + 1, _abi.ERR_LAYOUT), ("x.stride[3]", 2, _abi.ERR_LAYOUT),
        ("x.stride[1]", -1, _abi.ERR_LAYOUT), ("weight", FAKE + 2, _abi.ERR_LAYOUT), ("stats", FAKE + 4, _abi.ERR_LAYOUT)]


@pytest.mark.parametrize("path, value, code", NORM + [("eps", -1.0, _sln_abi.ERR_EPS), ("eps", float("nan"), _sln_abi.ERR_EPS), ("eps", float("inf"), _sln_abi.ERR_EPS),
                                                      ("y.data", None, _abi.ERR_NULL_POINTER), ("bias", FAKE + 1, _abi.ERR_LAYOUT)])
def test_norm_forward_refuses(path, value, code):
    a = fwd()
    assert lib().sln_validate_fwd(ctypes.byref(a)) == _abi.OK
    put(path, value)(a)
    assert lib().sln_validate_fwd(ctypes.byref(a)) == lib().sln_fwd(ctypes.byref(a), None) == code


@pytest.mark.parametrize("path, value, code", NORM + [
    ("stats", None, _abi.ERR_NULL_POINTER), ("dy.data", None, _abi.ERR_NULL_POINTER), ("dx.stride[3]", 0, _abi.ERR_LAYOUT),
    ("dweight", FAKE + 2, _abi.ERR_LAYOUT), ("dbias", FAKE + 1, _abi.ERR_LAYOUT), ("workspace", None, _abi.ERR_WORKSPACE),
    ("workspace", FAKE + 4, _abi.ERR_WORKSPACE), ("workspace_bytes", 8, _abi.ERR_WORKSPACE)])
def test_norm_backward_refuses(path, value, code):
    a = bwd()
    assert a.workspace_bytes and lib().sln_validate_bwd(ctypes.byref(a)) == _abi.OK
    put(path, value)(a)
    assert lib().sln_validate_bwd(ctypes.byref(a)) == lib().sln_bwd(ctypes.byref(a), None) == code


def test_norm_workspaces():
    a = bwd()
    a.dweight = a.dbias = None
    assert lib().sln_bwd_workspace_bytes(ctypes.byref(a)) == 0
    a.workspace = a.dx.data = None  # neither is used then
    assert lib().sln_validate_bwd(ctypes.byref(a)) == _abi.OK
    a = bwd()
    a.rows = 10  # one workgroup takes them all
    assert lib().sln_bwd_workspace_bytes(ctypes.byref(a)) == lib().sln_bwd_workspace_bytes(None) == 0


def test_error_strings():
    for name in ABIS:
        text = getattr(lib(), f"{name}_error_string")
        codes = (_spa_abi.ERR_PAGES, _spa_abi.ERR_ROWS) if name == "spa" else (_sln_abi.ERR_WIDTH, _sln_abi.ERR_EPS)
        for code in (*codes, _abi.ERR_LAYOUT, _abi.ERR_ABI, _abi.ERR_DTYPE, _sda_abi.ERR_HEADS, _abi.ERR_WORKSPACE):
            assert text(code) and text(code) != text(-9999)
