"""The host code of the paged cache (tda_amd/csrc/spa_host.cpp) and of the layer norm (tda_amd/csrc/sln_host.cpp) built with
g++ under AddressSanitizer and UndefinedBehaviorSanitizer, with launchers that record what they get in place of the
kernels, and driven through rejections, extreme sizes and strides, the buffer sizes and the parameter blocks
(tests/sanitize/spa_driver.cpp).  CPU only."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SAN = os.path.join(ROOT, "tests", "sanitize")
CSRC = os.path.join(ROOT, "tda_amd", "csrc")


def test_host_abi_under_asan_ubsan(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ missing")
    exe = tmp_path / "spa_driver"
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
           "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           *[os.path.join(CSRC, f) for f in ("spa_host.cpp", "sln_host.cpp", "sda_host.cpp", "tda_host.cpp")],
           os.path.join(SAN, "stub_launch.cpp"), os.path.join(SAN, "spa_driver.cpp"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all checks passed" in r.stdout
