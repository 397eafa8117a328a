"""What surrounds the 8-bit linear path on the host, without a GPU: the helpers of kd_host.h and the Python operand's
refusals."""
import os
import shutil
import subprocess

import pytest
import torch

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


def test_weight_elsewhere_is_refused(kd):
    """A weight in host memory, or on another GPU than the context's, is turned away before the library is called."""
    ctx = object.__new__(kd.Context)  # (no GPU here: what checks arguments needs only the device's index)
    ctx.handle, ctx.device = None, 0
    out = kd.Fp8Rows.empty(32, 64, device="cpu")
    out.device = 0
    w = kd.KdLinear.of(torch.zeros(32, 68, dtype=torch.uint8), kd.Q8_0, 64, 32)
    assert w.device == -1 and kd.KdLinear().device is None
    for device in (-1, 1):
        w.device = device
        with pytest.raises(ValueError):
            ctx.quantize_weight_fp8(w, out)


def test_operand_refuses_codes_of_another_format(kd):
    """One-byte types that are not e4m3 codes are not read as such."""
    codes, scales = torch.zeros(3, 112, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    for good in (torch.uint8, torch.float8_e4m3fn):
        assert kd.Fp8Rows(codes.view(good), scales, 100).codes.dtype == good
    for bad in (torch.float8_e5m2, torch.float8_e4m3fnuz, torch.int8, torch.bool):
        with pytest.raises(ValueError):
            kd.Fp8Rows(codes.view(bad), scales, 100)
