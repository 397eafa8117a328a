"""The 8-bit linear path on the GPU where it can go wrong beyond its common sizes: weights and scale bytes that no writer
of the library makes, the few-token product's ring when it is used again, sums written in place by several warps,
captured runs beside other work, outputs that overlap themselves.  Tolerances are those of test_gpu_fp8.py."""
import numpy as np
import pytest
import torch

import fp8_ref
from helpers import seeded
from test_gpu_fp8 import HALF, TORCH, check_product, dev, f64, hidden, operand, rows_of

pytestmark = pytest.mark.gpu


def ggml_rows(name, codes, d):
    """Whole codes (C, K) under f16 scales (C, K / 32) as ggml blocks: (bytes, float64 values)."""
    C, K = codes.shape
    q = codes.reshape(C, K // 32, 32)
    if name == "q8_0":
        b = q.astype(np.int8).view(np.uint8)
    else:
        n = (q + 8).astype(np.uint8)
        b = n[:, :, :16] | (n[:, :, 16:] << 4)
    raw = np.concatenate([d[:, :, None].view(np.uint8).reshape(C, K // 32, 2), b], 2).reshape(C, -1)
    with np.errstate(invalid="ignore"):
        v = (d[:, :, None].astype(np.float64) * q).reshape(C, K)
    return np.ascontiguousarray(raw), v


@pytest.mark.parametrize("name", ["q8_0", "q4_0"])
@pytest.mark.parametrize("K", [32, 96, 256, 1056])
def test_ggml_zero_codes_under_any_scale(ctx, kd, name, K):
    """Blocks whose codes are all zero are zeros whatever their finite scale, alone, as a whole group of 128 columns and
    beside other blocks of the group; NaN under a scale that is not finite."""
    scales = [4.0, -4.0, 100.0, 65504.0, -65504.0, 3.9, 6e-8, 0.0]
    C = 2 * len(scales) + 2
    rng = np.random.default_rng(K)
    codes = rng.integers(-7, 8, (C, K))
    d = np.full((C, K // 32), 0.01, np.float16)
    for i, s in enumerate(scales):
        codes[2 * i] = 0                    # a whole row
        d[2 * i] = s
        codes[2 * i + 1, :32] = 0           # one block of a group
        d[2 * i + 1, 0] = s
    codes[C - 2:, :32] = 0
    d[C - 2, 0], d[C - 1, 0] = np.inf, np.nan
    raw, v = ggml_rows(name, codes, d)
    want, s = fp8_ref.encode(v)
    r = kd.Fp8Rows.empty(C, K)
    ctx.quantize_weight_fp8(kd.KdLinear.of(torch.from_numpy(raw).cuda(), kd.Q8_0 if name == "q8_0" else kd.Q4_0, K, C), r)
    got, gs = rows_of(r)
    assert np.array_equal(gs, s)
    assert np.array_equal(fp8_ref.VALUES[got], fp8_ref.VALUES[want], equal_nan=True)
    assert not np.isnan(fp8_ref.VALUES[got[:C - 2]]).any()
