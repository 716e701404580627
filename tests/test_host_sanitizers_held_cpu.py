"""The checks of place with counts of held pages under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only); see tests/host_sanitizer_held_driver.cpp."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT


def test_argument_checks_are_sanitizer_clean(tmp_path):
    rocm = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
    if shutil.which("g++") is None or not (rocm / "include" / "hip").exists():
        pytest.skip("g++ or HIP's headers not available")
    exe, csrc = tmp_path / "drv", ROOT / "cudalab_amd" / "csrc"
    build = subprocess.run(
        ["g++", "-std=c++20", "-O1", "-g", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
         "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         f"-I{rocm / 'include'}", f"-I{ROOT / 'include'}", f"-I{csrc}",
         str(csrc / "cq_place_capi.cpp"), str(ROOT / "tests" / "host_sanitizer_held_driver.cpp"),
         "-o", str(exe), f"-L{rocm / 'lib'}", "-lamdhip64", f"-Wl,-rpath,{rocm / 'lib'}"],
        capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-3000:]
    assert "runtime error" not in out and out.rstrip().endswith("done"), out[-3000:]
