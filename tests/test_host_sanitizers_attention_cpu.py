"""The host code of the calls around attention under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only), over sizes, strides and pointers at the
ends of their types; see tests/host_sanitizer_attention_driver.cpp."""
from __future__ import annotations

import os
import shlex
import subprocess

import pytest

from test_host_sanitizers_cpu import ROOT, SANITIZE, _hipcc


def test_attention_host_code_is_sanitizer_clean(tmp_path):
    hipcc = _hipcc()
    if hipcc is None:
        pytest.skip("hipcc not available")
    exe = tmp_path / "drv"
    csrc = ROOT / "cudalab_amd" / "csrc"
    flags = ["--offload-arch=gfx950", "-O1", "-g", "-std=c++20", "-Xclang", "-target-feature",
             "-Xclang", "-packed-fp32-ops", *shlex.split(SANITIZE),
             "-I", str(ROOT / "include"), "-I", str(csrc)]
    files = [csrc / n for n in ("cq_capi.cpp", "cq_attn_capi.cpp", "cq_kernels.hip",
                                "cq_quantize.hip", "cq_norm_rope.hip", "cq_kvcache.hip",
                                "cq_attention.hip")]
    files.append(ROOT / "tests" / "host_sanitizer_attention_driver.cpp")
    jobs = [subprocess.Popen([hipcc, *flags, "-c", str(f), "-o", str(tmp_path / f"{f.stem}.o")],
                             stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
            for f in files]
    for j in jobs:
        out, _ = j.communicate(timeout=600)
        assert j.returncode == 0, out[-2000:]
    link = subprocess.run([hipcc, "--offload-arch=gfx950", *shlex.split(SANITIZE),
                           *(str(tmp_path / f"{f.stem}.o") for f in files), "-o", str(exe)],
                          capture_output=True, text=True, timeout=600)
    assert link.returncode == 0, link.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-3000:]
    assert "ERROR: AddressSanitizer" not in out and "runtime error" not in out, out[-3000:]
    assert "refused some, planned some, wrong 0" in out and out.rstrip().endswith("done")
