"""8-bit rows without a GPU: the scale-tile size, the Python operand's checks, the tensor core's block-scaled
descriptors against CUTLASS's bit fields, and the tests' own 64-bit restatement."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import fp8_ref
from test_descriptors import ROOT, cutlass_include


def test_block_scaled_descriptors_match_cutlass(tmp_path):
    inc = cutlass_include()
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if inc is None or not os.path.exists(nvcc):
        pytest.skip("CUTLASS headers or nvcc not available")
    exe = str(tmp_path / "desc8_check")
    r = subprocess.run([nvcc, "-std=c++17", "-I", inc, "-I", os.path.join(ROOT, "kandinsky.cpp_b200", "csrc"),
                        "-o", exe, os.path.join(ROOT, "tests", "native", "desc8_check.cu")], capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr


@pytest.mark.parametrize("K,rows,want", [(1, 1, 512), (512, 128, 512), (513, 128, 1024), (512, 129, 1024),
                                         (4096, 31744, 248 * 8 * 512), (128, 0, 0)])
def test_scale_bytes(kd, K, rows, want):
    assert kd.fp8_scale_bytes(K, rows) == want
    if rows:
        assert fp8_ref.tile_offsets(rows, K).max() < want
        assert np.unique(fp8_ref.tile_offsets(rows, K)).size == rows * -(-K // 128)


@pytest.mark.parametrize("K,rows", [(0, 1), (-5, 1), (128, -1), ((1 << 20) + 1, 1), (128, (1 << 24) + 1)])
def test_scale_bytes_refuses(kd, K, rows):
    with pytest.raises(kd.KdAttnError):
        kd.fp8_scale_bytes(K, rows)


def test_operand_checks(kd):
    codes = torch.zeros(3, 112, dtype=torch.uint8)
    scales = torch.zeros(512, dtype=torch.uint8)
    r = kd.Fp8Rows(codes, scales, 100)
    assert (r.rows, r.in_features, r.struct.nb1, list(r.struct.ne)) == (3, 100, 112, [100, 3])
    for bad in ((codes.float(), scales, 100), (codes.t(), scales, 100), (codes[0], scales, 100),
                (codes, scales, 113), (codes, scales[:511], 100), (codes, scales.float(), 100)):
        with pytest.raises(ValueError):
            kd.Fp8Rows(*bad)
    e = kd.Fp8Rows.empty(5, 130, device="cpu")
    assert tuple(e.codes.shape) == (5, 256) and e.scales.numel() == 512 and e.codes.dtype == torch.float8_e4m3fn


def test_entry_points_refuse_a_null_context(kd):
    L = kd.lib
    assert L.kd_attn_quantize_fp8(None, None, None, None) == kd.ERR_INVALID_ARGUMENT
    assert L.kd_attn_quantize_weight_fp8(None, None, None, None) == kd.ERR_INVALID_ARGUMENT
    assert L.kd_attn_dequantize_fp8(None, None, None, None) == kd.ERR_INVALID_ARGUMENT
    assert L.kd_attn_rms_norm_fp8(None, None, None, None, 1e-6, None, None, None) == kd.ERR_INVALID_ARGUMENT
    assert L.kd_attn_linear_fp8(None, None, None, None, None, None) == kd.ERR_INVALID_ARGUMENT


def test_reference_restatement_agrees_with_torch():
    """The tests' e4m3 rounding against torch's cast, ties and subnormals among the values."""
    v = np.concatenate([np.linspace(-448, 448, 20011), np.arange(-64, 65) / 1024.0,
                        (fp8_ref.VALUES[:126] + fp8_ref.VALUES[1:127]) / 2])
    want = torch.from_numpy(v).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    got = fp8_ref.round_e4m3(v.astype(np.float32).astype(np.float64))
    assert np.array_equal(fp8_ref.VALUES[got], fp8_ref.VALUES[want])


def build_host_test(kd, tmp_path):
    """g++ -> tests/native/host_fp8_test linked against libkd_attn.so and cudart."""
    gxx, cuda = shutil.which("g++"), os.environ.get("CUDA_HOME", "/usr/local/cuda")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "host_fp8_test")
    lib_dir, rt = os.path.dirname(kd.LIB_PATH), os.path.join(cuda, "lib64")
    cmd = [gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(ROOT, "kandinsky.cpp_b200", "host"), "-I", os.path.join(cuda, "include"),
           os.path.join(ROOT, "tests", "native", "host_fp8_test.cpp"), "-o", exe, kd.LIB_PATH, "-L", rt, "-lcudart",
           f"-Wl,-rpath,{lib_dir}", f"-Wl,-rpath,{rt}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return exe


def test_host_layer_on_cpu(kd, tmp_path):
    out = subprocess.run([build_host_test(kd, tmp_path), "--cpu"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr


@pytest.mark.gpu
def test_host_layer_on_gpu(kd, tmp_path):
    out = subprocess.run([build_host_test(kd, tmp_path)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip().endswith("OK"), out.stdout + out.stderr
