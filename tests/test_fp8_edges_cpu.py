"""What surrounds the 8-bit linear path on the host, without a GPU: the helpers of kd_host.h and the Python operand's
refusals."""
import os
import shutil
import subprocess

import pytest

from test_descriptors import ROOT


def test_host_helpers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "host_util_check")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "kandinsky.cpp_b200", "csrc"),
                        os.path.join(ROOT, "tests", "native", "host_util_check.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr
