"""The 8-bit linear path on the GPU against the 64-bit restatement in fp8_ref.py.

Tolerances: quantising and reading back round once, so codes, scale bytes and values are compared bit for bit.  The
norm computes v in f32 before it rounds to e4m3: each value is off v by at most half an e4m3 step (2^-4 of it, or
2^-10 of the block's scale for subnormal codes) and the f32 error of v, which a sum of K squares in f32 bounds by
(K / 2 + 8) * 2^-24 of it (half of the sum's relative error, and the rest of the chain); its scale is that of the
f32 maximum.  The product's terms are exact in f32 (4 x 4 significant bits); summing K of them in f32 in any order,
truncated or rounded, is off by at most K * 2^-23 * sum |x w|, and the output rounds once: half a step, 2^-p of
the value with p significant bits, or 2^-25 where it is below f16's smallest normal number 2^-14 (steps of 2^-24)."""
import numpy as np
import pytest
import torch

import fp8_ref
import oracle
from helpers import seeded

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def hidden(R, K, seed):
    """Normal values; every 50th column is large and every 7th block of a row small, so that scales differ."""
    v = seeded((R, K), seed, 0).astype(np.float32)
    v[:, ::50] *= 30.0
    for b in range(0, K, 128):
        v[(b // 128) % 7::7, b:b + 128] *= 1e-3
    return v


def dev(a, dtype="f32"):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().to(TORCH[dtype])


def f64(t):
    return t.double().cpu().numpy()


def rows_of(r):
    """(codes, scale bytes) of an Fp8Rows on the host."""
    codes = r.codes.view(torch.uint8).cpu().numpy()[:, :r.in_features]
    return codes, r.scales.cpu().numpy()[fp8_ref.tile_offsets(r.rows, r.in_features)]


def operand(kd, v):
    """An Fp8Rows of float64 rows, laid out by the restatement; what lies outside the rows is poisoned (codes past
    K and scale bytes of no row are NaN)."""
    codes, s = fp8_ref.encode(v)
    R, K = codes.shape
    r = kd.Fp8Rows.empty(R, K)
    c = np.full((R, r.codes.shape[1]), 0x7F, np.uint8)
    c[:, :K] = codes
    t = np.full(r.scales.numel(), 0xFF, np.uint8)
    t[fp8_ref.tile_offsets(R, K)] = s
    r.codes.view(torch.uint8).copy_(torch.from_numpy(c))
    r.scales.copy_(torch.from_numpy(t))
    return r, fp8_ref.decode(codes, s)


# ------------------------------------------------------------------ quantise / read back
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 128), (3, 129), (33, 777), (130, 512), (257, 520), (40, 4096)])
def test_quantize_and_read_back(ctx, kd, R, K, dtype):
    x = dev(hidden(R, K, 11), dtype)
    codes, s = fp8_ref.encode(f64(x))
    r = kd.Fp8Rows.empty(R, K)
    ctx.quantize_fp8(x, r)
    got, gs = rows_of(r)
    assert np.array_equal(gs, s)
    assert np.array_equal(got, codes)
    for out in ("f32", "f16", "bf16"):
        y = torch.full((R, K), float("nan"), device="cuda", dtype=TORCH[out])
        ctx.dequantize_fp8(r, y)
        assert np.array_equal(f64(y), fp8_ref.round_to(fp8_ref.decode(codes, s), out))


def test_quantize_strided_and_misaligned(ctx, kd):
    """[K, L, N] views: rows of a wider buffer, an odd start, tokens and sequences exchanged."""
    N, L, K = 3, 5, 300
    wide = dev(hidden(N * L, 2 * K + 7, 12), "bf16").view(N, L, -1)
    for x in (wide[:, :, :K], wide[:, :, 3:3 + K], wide[:, :, K:2 * K].transpose(0, 1), wide[1, :, 1:1 + K],
              wide[:1, :1, 5:5 + K].expand(2, 4, K)):
        rows = x.numel() // K
        codes, s = fp8_ref.encode(f64(x).reshape(rows, K))
        r = kd.Fp8Rows.empty(rows, K)
        ctx.quantize_fp8(x, r)
        got, gs = rows_of(r)
        assert np.array_equal(gs, s) and np.array_equal(got, codes)
        y = torch.full((N, L, 2 * K + 7), 7.0, device="cuda")
        if x.shape == (N, L, K):
            ctx.dequantize_fp8(r, y[:, :, 3:3 + K])
            assert np.array_equal(f64(y[:, :, 3:3 + K]).reshape(rows, K), fp8_ref.decode(codes, s).astype(np.float32))
            assert (y[:, :, :3] == 7).all() and (y[:, :, 3 + K:] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("K", [1, 2, 63, 129, 511, 512, 513, 1023, 1025, 1537])
def test_rows_that_start_anywhere(ctx, kd, K, dtype):
    """Quantising, the norm with residual and h, and reading back, on rows that start on every residue of 16 bytes."""
    R = 9
    for start, pad in ((0, 1), (1, 0), (1, 1), (3, 2), (2, 4)):
        def place(v):
            wide = torch.full((R, start + K + pad), 5.0, device="cuda", dtype=TORCH[dtype])
            wide[:, start:start + K] = v
            return wide, wide[:, start:start + K]
        _, x = place(dev(hidden(R, K, 14), dtype))
        _, res = place(dev(seeded((R, K), 15, 0), dtype))
        r = kd.Fp8Rows.empty(R, K)
        ctx.quantize_fp8(x, r)
        codes, s = fp8_ref.encode(f64(x))
        got, gs = rows_of(r)
        assert np.array_equal(gs, s) and np.array_equal(got, codes)
        wy, y = place(0.0)
        ctx.dequantize_fp8(r, y)
        assert np.array_equal(f64(y), fp8_ref.round_to(fp8_ref.decode(codes, s), dtype))
        wh, h = place(0.0)
        ctx.rms_norm_fp8(x, r, residual=res, h=h)
        assert torch.equal(h, (x.float() + res.float()).to(TORCH[dtype]))
        check_norm(kd, r, f64(h), None, 1e-6)
        for w in (wy, wh):
            assert (w[:, :start] == 5).all() and (w[:, start + K:] == 5).all()


def test_quantize_edges(ctx, kd):
    """Zeros, the scale's border (448 * 2^e and one step above), subnormal inputs, NaN and infinities; codes and
    scales outside the rows stay as they were."""
    K = 256
    v = np.zeros((8, K), np.float32)
    v[1, :] = 448.0
    v[2, 5] = np.nextafter(np.float32(448.0), np.float32(1e9))
    v[3, :] = 1e-42
    v[4, 10], v[4, 11], v[4, 12], v[4, 13] = np.nan, np.inf, -np.inf, 3.0
    v[5, 200] = np.float32(3.4e38)
    v[6, :] = np.linspace(-1, 1, K, dtype=np.float32)
    v[7, 0] = -0.0
    codes, s = fp8_ref.encode(v.astype(np.float64))
    r = kd.Fp8Rows.empty(8, K)
    r.codes.view(torch.uint8).fill_(0xAA)
    r.scales.fill_(0xBB)
    part = kd.Fp8Rows(r.codes[:8], r.scales, K)
    ctx.quantize_fp8(dev(v), part)
    got, gs = rows_of(part)
    assert np.array_equal(gs, s)
    assert np.array_equal(fp8_ref.VALUES[got], fp8_ref.VALUES[codes], equal_nan=True)
    left = np.ones(r.scales.numel(), bool)
    left[fp8_ref.tile_offsets(8, K)] = False
    assert (r.scales.cpu().numpy()[left] == 0xBB).all()
    y = torch.empty(8, K, device="cuda")
    ctx.dequantize_fp8(part, y)
    y = y.cpu().numpy()
    assert np.isnan(y[4, 10:13]).all() and y[4, 13] == 3.0 and (y[0] == 0).all() and y[2, 5] == 448.0


@pytest.mark.parametrize("name", ["q8_0", "q4_0", "f16", "bf16", "f32"])
@pytest.mark.parametrize("C,K", [(5, 32), (64, 416), (129, 1024), (33, 4096), (7, 1536), (9, 2080)])
def test_quantize_weight(ctx, kd, name, C, K):
    w = (seeded((C, K), 13, 0) / np.sqrt(K)).astype(np.float32)
    wtype = {"q8_0": kd.Q8_0, "q4_0": kd.Q4_0, "f16": kd.F16, "bf16": kd.BF16, "f32": kd.F32}[name]
    if name in ("q8_0", "q4_0"):
        raw = oracle.quantize_q8_0(w) if name == "q8_0" else oracle.quantize_q4_0(w)
        deq = oracle.dequantize(raw, wtype, K)
        t = torch.from_numpy(raw).cuda()
    else:
        t = dev(w, name)
        deq = f64(t)
    r = kd.Fp8Rows.empty(C, K)
    ctx.quantize_weight_fp8(kd.KdLinear.of(t, wtype, K, C), r)
    codes, s = fp8_ref.encode(np.asarray(deq, np.float64))
    got, gs = rows_of(r)
    assert np.array_equal(gs, s)
    # a ggml zero may be -0 * d
    assert np.array_equal(fp8_ref.VALUES[got], fp8_ref.VALUES[codes])


def test_quantize_ggml_edges(ctx, kd):
    """ggml blocks with scales of zero, negative, subnormal, infinite and NaN, and the extreme codes."""
    K, C = 256, 6
    raw = np.zeros((C, K // 32, 34), np.uint8)
    raw[:, :, 2:] = np.arange(32, dtype=np.uint8) * 8 + np.arange(K // 32, dtype=np.uint8)[:, None]  # all of int8 among them
    d = np.full((C, K // 32), 0.01, np.float16)
    d[0, 1], d[1, :4], d[2, 2], d[3, 5], d[4, 6] = -0.5, 0.0, 6e-8, np.inf, np.nan
    raw[:, :, :2] = d.view(np.uint8).reshape(C, K // 32, 2)
    with np.errstate(invalid="ignore"):
        v = (d[:, :, None].astype(np.float64) * raw[:, :, 2:].view(np.int8)).reshape(C, K)
    codes, s = fp8_ref.encode(v)
    r = kd.Fp8Rows.empty(C, K)
    t = torch.from_numpy(raw.reshape(C, -1)).cuda()
    ctx.quantize_weight_fp8(kd.KdLinear.of(t, kd.Q8_0, K, C), r)
    got, gs = rows_of(r)
    assert np.array_equal(gs, s)
    assert np.array_equal(fp8_ref.VALUES[got], fp8_ref.VALUES[codes], equal_nan=True)


# ------------------------------------------------------------------ norm
def check_norm(kd, r, h64, gain, eps):
    v = h64 / np.sqrt(np.mean(h64 ** 2, axis=1, keepdims=True) + eps)
    if gain is not None:
        v = v * gain
    R, K = v.shape
    err = (K / 2 + 8) * 2.0 ** -24
    codes, gs = rows_of(r)
    nb = gs.shape[1]
    p = np.zeros((R, nb * 128))
    p[:, :K] = np.abs(v)
    top = p.reshape(R, nb, 128).max(2)
    e = gs.astype(np.float64) - 127
    assert (top * (1 - err) <= 448 * 2.0 ** e).all()
    assert ((top * (1 + err) > 448 * 2.0 ** (e - 1)) | (gs == 1)).all()
    got = fp8_ref.decode(codes, gs)
    step = np.repeat(2.0 ** e, 128, axis=1)[:, :K]
    assert (np.abs(got - v) <= np.maximum(np.abs(v) * 2.0 ** -4, step * 2.0 ** -10) + err * np.abs(v)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 4096), (3, 128), (5, 257), (130, 100), (77, 1000), (9, 1792), (4, 8193),
                                 (3, 16400), (2, 32768)])
def test_norm(ctx, kd, R, K, dtype):
    x, res = dev(hidden(R, K, 21), dtype), dev(seeded((R, K), 22, 0), dtype)
    gain = (1 + 0.1 * seeded((K,), 23, 0)).astype(np.float32)
    s64 = fp8_ref.round_to(f64(x) + f64(res), dtype)
    for use_res in (True, False):
        r = kd.Fp8Rows.empty(R, K)
        h = torch.full_like(x, float("nan"))
        ctx.rms_norm_fp8(x, r, residual=res if use_res else None, gain=dev(gain), h=h)
        h64 = f64(h)
        if use_res:
            # x + res in f32 and then in the rows' type: within one more rounding of the sum rounded once
            assert (np.abs(h64 - s64) <= 2 * HALF[dtype] * np.abs(s64) + (2.0 ** -24 if dtype == "f16" else 0) + 2.0 ** -24 * (np.abs(f64(x)) + np.abs(f64(res)))).all()
        else:
            assert torch.equal(h, x)
        check_norm(kd, r, h64, gain.astype(np.float64), 1e-6)
        q = kd.Fp8Rows.empty(R, K)  # without h the same rows come out
        ctx.rms_norm_fp8(x, q, residual=res if use_res else None, gain=dev(gain))
        assert all(np.array_equal(a, b) for a, b in zip(rows_of(r), rows_of(q)))


def test_norm_strided_in_place_and_edges(ctx, kd):
    """Views with tokens and sequences exchanged, the sum written over x and over the residual, unit gain, a row of
    zeros, tiny rows that eps decides, and a row with a NaN, which alone is NaN."""
    N, L, K = 2, 6, 200
    base = dev(hidden(N * L, K, 24)).view(N, L, K)
    base[0, 1] = 0
    base[0, 2] *= 1e-6
    base[1, 3, 17] = float("nan")
    x = base.transpose(0, 1)                       # [K, N, L]: tokens and sequences exchanged
    res = dev(seeded((L, N, K + 4), 25, 0))[:, :, 4:]
    res[1, 0] = 0
    want = f64(x + res).reshape(N * L, K)
    clean = ~np.isnan(want).any(1)
    for target in ("x", "res", "new"):
        xi, ri = x.clone(memory_format=torch.preserve_format), res.clone()
        h = xi if target == "x" else ri if target == "res" else torch.empty(L, N, K, device="cuda")
        r = kd.Fp8Rows.empty(N * L, K)
        ctx.rms_norm_fp8(xi, r, residual=ri, eps=1e-5, h=h)
        assert np.array_equal(f64(h).reshape(N * L, K), want, equal_nan=True)
        codes, gs = rows_of(r)
        assert np.isnan(fp8_ref.VALUES[codes[~clean]]).all() and (~clean).sum() == 1
        q = kd.Fp8Rows.empty(int(clean.sum()), K)
        ctx.rms_norm_fp8(h.reshape(N * L, K)[torch.from_numpy(clean).cuda()], q, eps=1e-5)
        qc, qs = rows_of(q)
        assert np.array_equal(codes[clean], qc) and np.array_equal(gs[clean], qs)
        check_norm(kd, q, want[clean], None, 1e-5)
        zero = codes[~np.any(want, axis=1)]
        assert zero.shape[0] == 1 and not (zero & 0x7F).any()


# ------------------------------------------------------------------ product
def check_product(y, x64, w64, bias, dtype, label=""):
    want = x64 @ w64.T + (0 if bias is None else bias)
    room = np.abs(x64) @ np.abs(w64).T + (0 if bias is None else np.abs(bias))
    err = np.abs(f64(y).reshape(want.shape) - want)
    lim = HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0) + (x64.shape[1] + 1) * 2.0 ** -23 * room
    worst = float(np.max(err / np.maximum(lim, 1e-300)))
    assert worst <= 1, f"{label}: {worst:.3g} of the bound"
    return float(np.linalg.norm(err) / max(np.linalg.norm(want), 1e-300))


SIZES = [(1, 1, 1), (1, 128, 128), (2, 130, 16), (1, 1000, 4096), (16, 256, 512), (17, 100, 200), (33, 129, 640),
         (77, 384, 1000), (128, 128, 1152), (129, 384, 520), (256, 200, 2048), (257, 300, 640), (600, 520, 1792),
         (1030, 256, 130), (3000, 1152, 300), (4608, 1000, 520), (4608, 1536, 640),
         (300, 28416, 128), (20000, 384, 256), (20000, 384, 384), (9500, 1100, 96), (9500, 576, 300),
         (20000, 256, 640)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(ctx, kd, M, N, K, dtype):
    x, x64 = operand(kd, hidden(M, K, 31))
    w, w64 = operand(kd, hidden(N, K, 32) / np.sqrt(K))
    bias = seeded((N,), 33, 0).astype(np.float32)
    for b in (bias, None):
        y = torch.full((M + 1, N), 5.0, device="cuda", dtype=TORCH[dtype])
        ctx.linear_fp8(x, w, y[:M], bias=None if b is None else dev(b))
        ctx.device_status()
        check_product(y[:M], x64, w64, b, dtype, f"{M}x{N}x{K}")
        assert (y[M] == 5).all()


def test_linear_strided_output(ctx, kd):
    """y as rows of a wider buffer, at an odd column, with tokens and sequences exchanged, and a misaligned bias."""
    N, L, C, K = 3, 50, 200, 384
    x, x64 = operand(kd, hidden(N * L, K, 34))
    w, w64 = operand(kd, hidden(C, K, 35) / np.sqrt(K))
    bias = dev(seeded((C + 1,), 36, 0))[1:]
    for dtype in ("bf16", "f32"):
        for odd in (0, 1):
            wide = torch.full((N, L, C + 24), 3.0, device="cuda", dtype=TORCH[dtype])
            y = wide[:, :, odd:odd + C]
            ctx.linear_fp8(x, w, y, bias=bias)
            check_product(y.reshape(N * L, C), x64, w64, f64(bias), dtype)
            assert (wide[:, :, :odd] == 3).all() and (wide[:, :, odd + C:] == 3).all()
        t = torch.full((L, N, C), 3.0, device="cuda", dtype=TORCH[dtype])
        ctx.linear_fp8(x, w, t.transpose(0, 1), bias=bias)
        check_product(t.transpose(0, 1).reshape(N * L, C), x64, w64, f64(bias), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C", [1, 63, 130, 193, 383, 577])
def test_linear_many_tokens_rows_anywhere(ctx, kd, C, dtype):
    """More tokens than one tile into rows that start on every residue of 32 bytes, odd widths, two sequences."""
    N, L, K = 2, 333, 200
    x, x64 = operand(kd, hidden(N * L, K, 61))
    w, w64 = operand(kd, hidden(C, K, 62) / np.sqrt(K))
    bias = dev(seeded((C,), 63, 0))
    for start, pad in ((0, 0), (1, 3), (2, 6), (3, 5), (0, 1)):
        wide = torch.full((N, L + 1, start + C + pad), 9.0, device="cuda", dtype=TORCH[dtype])
        y = wide[:, :L, start:start + C]
        ctx.linear_fp8(x, w, y, bias=bias)
        check_product(y.reshape(N * L, C), x64, w64, f64(bias), dtype, f"C {C} start {start} pad {pad}")
        assert (wide[:, :, :start] == 9).all() and (wide[:, :, start + C:] == 9).all() and (wide[:, L] == 9).all()


def test_linear_nan_stays_in_its_row(ctx, kd):
    M, N, K = 40, 256, 512
    x, x64 = operand(kd, hidden(M, K, 37))
    w, w64 = operand(kd, hidden(N, K, 38))
    x.codes.view(torch.uint8)[7, 300] = 0x7F
    y = torch.empty(M, N, device="cuda")
    ctx.linear_fp8(x, w, y)
    bad = torch.isnan(y).any(1).cpu().numpy()
    assert bad[7] and bad.sum() == 1 and torch.isnan(y[7]).all()
    keep = np.arange(M) != 7
    check_product(y[torch.from_numpy(keep).cuda()], x64[keep], w64, None, "f32")


def test_linear_same_bits_every_time(ctx, kd):
    M, N, K = 20, 640, 4096
    x, _ = operand(kd, hidden(M, K, 39))
    w, _ = operand(kd, hidden(N, K, 40))
    ys = [ctx.linear_fp8(x, w, torch.empty(M, N, device="cuda")) for _ in range(5)]
    assert all(torch.equal(ys[0], y) for y in ys[1:])


def test_run_as_used(ctx, kd):
    """Norm with the residual, a widening product, its output quantised, a narrowing product: the pieces together
    against the same steps in 64 bits on the values that the 8-bit rows hold."""
    N, L, C, F = 2, 75, 512, 1024
    x, res = dev(hidden(N * L, C, 41), "bf16").view(N, L, C), dev(seeded((N, L, C), 42, 0), "bf16")
    gain = dev(1 + 0.1 * seeded((C,), 43, 0))
    ws = []
    for i, (o, k) in enumerate(((F, C), (C, F))):
        wt = (seeded((o, k), 44, i) / np.sqrt(k)).astype(np.float32)
        raw = oracle.quantize_q8_0(wt)
        r = kd.Fp8Rows.empty(o, k)
        ctx.quantize_weight_fp8(kd.KdLinear.of(torch.from_numpy(raw).cuda(), kd.Q8_0, k, o), r)
        ws.append(r)
    h, a, b = torch.empty_like(x), kd.Fp8Rows.empty(N * L, C), kd.Fp8Rows.empty(N * L, F)
    up, y = torch.empty(N, L, F, device="cuda", dtype=torch.bfloat16), torch.empty(N, L, C, device="cuda")
    ctx.rms_norm_fp8(x, a, residual=res, gain=gain, h=h)
    ctx.linear_fp8(a, ws[0], up)
    ctx.quantize_fp8(up, b)
    ctx.linear_fp8(b, ws[1], y)
    ctx.device_status()
    check_norm(kd, a, f64(h).reshape(N * L, C), f64(gain), 1e-6)
    vals = [fp8_ref.decode(*rows_of(r)) for r in (a, b, *ws)]
    check_product(up, vals[0], vals[2], None, "bf16")
    codes, s = fp8_ref.encode(f64(up).reshape(N * L, F))
    assert all(np.array_equal(p, q) for p, q in zip(rows_of(b), (codes, s)))
    check_product(y, vals[1], vals[3], None, "f32")


def test_streams_and_graph(ctx, kd):
    """The run on a side stream and captured into a graph that is replayed on new inputs."""
    M, C, F = 50, 384, 640
    x = dev(hidden(M, C, 51), "bf16")
    w, w64 = operand(kd, hidden(F, C, 52))
    a, y = kd.Fp8Rows.empty(M, C), torch.empty(M, F, device="cuda")

    def run():
        ctx.rms_norm_fp8(x, a)
        ctx.linear_fp8(a, w, y)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    check_product(y, fp8_ref.decode(*rows_of(a)), w64, None, "f32")
    first = y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    y.zero_()
    g.replay()
    assert torch.equal(y, first)
    x.copy_(dev(hidden(M, C, 53), "bf16"))
    g.replay()
    check_product(y, fp8_ref.decode(*rows_of(a)), w64, None, "f32")
    assert not torch.equal(y, first)
    ctx.device_status()


def test_back_to_back(ctx, kd):
    """Launches that may overlap the one before: a chain whose every step reads what the last wrote and writes what the
    one before read, over buffers used again at once, gives what the same chain gives with a wait after every call."""
    M, C = 300, 640
    ws = [operand(kd, hidden(C, C, 70 + i) / np.sqrt(C))[0] for i in range(2)]
    x0 = dev(hidden(M, C, 72), "bf16")

    def chain(sync, m):
        x, y, h = x0[:m].clone(), torch.empty(m, C, device="cuda", dtype=torch.bfloat16), torch.empty(m, C, device="cuda", dtype=torch.bfloat16)
        a = kd.Fp8Rows.empty(m, C)
        for i in range(40):
            for call in (lambda: ctx.rms_norm_fp8(x, a, residual=y if i else None, h=h), lambda: ctx.linear_fp8(a, ws[i & 1], y),
                         lambda: ctx.quantize_fp8(y, a), lambda: ctx.linear_fp8(a, ws[1 - (i & 1)], x),
                         lambda: ctx.dequantize_fp8(a, h), lambda: x.add_(h)):
                call()
                if sync:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return x, y, h, *rows_of(a)

    for m in (3, 200, M):
        for p, q in zip(chain(False, m), chain(True, m)):
            assert torch.equal(p, q) if isinstance(p, torch.Tensor) else np.array_equal(p, q)
    ctx.device_status()


def test_empty(ctx, kd):
    e, w = kd.Fp8Rows.empty(0, 64), kd.Fp8Rows.empty(32, 64)
    ctx.quantize_fp8(torch.empty(0, 64, device="cuda"), e)
    ctx.rms_norm_fp8(torch.empty(0, 64, device="cuda"), e, h=torch.empty(0, 64, device="cuda"))
    ctx.dequantize_fp8(e, torch.empty(0, 64, device="cuda"))
    ctx.linear_fp8(e, w, torch.empty(0, 32, device="cuda"))
    ctx.device_status()


def test_refusals(ctx, kd):
    """What the host turns away, before any launch."""
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    r, w = kd.Fp8Rows.empty(4, 64), kd.Fp8Rows.empty(32, 64)

    def refused(call, status):
        with pytest.raises(kd.KdAttnError) as e:
            call()
        assert e.value.status == status and str(e.value)

    bad, uns = kd.ERR_INVALID_ARGUMENT, kd.ERR_UNSUPPORTED
    refused(lambda: ctx.quantize_fp8(z(5, 64), r), bad)                              # another number of rows
    refused(lambda: ctx.quantize_fp8(z(4, 65), r), bad)                              # columns
    refused(lambda: ctx.quantize_fp8(z(64, 4).t(), r), uns)                          # dim 0 not contiguous
    refused(lambda: ctx.dequantize_fp8(r, z(4, 63)), bad)
    refused(lambda: ctx.dequantize_fp8(r, z(1, 64).expand(4, 64)), bad)              # rows written over each other
    refused(lambda: ctx.rms_norm_fp8(z(4, 64), r, residual=z(4, 64, dtype=torch.float16)), bad)
    refused(lambda: ctx.rms_norm_fp8(z(4, 64), r, residual=z(2, 2, 64)), bad)
    refused(lambda: ctx.rms_norm_fp8(z(4, 64), r, h=z(1, 64).expand(4, 64)), bad)
    refused(lambda: ctx.rms_norm_fp8(z(4, 64), r, eps=-1.0), bad)
    refused(lambda: ctx.rms_norm_fp8(z(4, 64), r, eps=float("nan")), bad)
    wide = kd.Fp8Rows.empty(1, 32769)
    refused(lambda: ctx.rms_norm_fp8(z(1, 32769), wide), uns)
    refused(lambda: ctx.linear_fp8(r, kd.Fp8Rows.empty(32, 128), z(4, 32)), bad)     # K differs
    refused(lambda: ctx.linear_fp8(r, w, z(4, 33)), bad)
    refused(lambda: ctx.linear_fp8(r, w, z(32, 4).t()), uns)
    lin = kd.KdLinear.of(z(32, 64 // 32 * 34, dtype=torch.uint8), kd.Q8_0, 64, 32)
    refused(lambda: ctx.quantize_weight_fp8(lin, r), bad)
    odd = kd.Fp8Rows.empty(2, 48)
    refused(lambda: ctx.quantize_weight_fp8(kd.KdLinear.of(z(2, 34, dtype=torch.uint8), kd.Q8_0, 48, 2), odd), uns)
    refused(lambda: ctx.quantize_weight_fp8(kd.KdLinear.of(z(4, 64), 99, 64, 4), r), uns)
    pitch = kd.Fp8Rows(z(4, 72, dtype=torch.uint8), r.scales, 64)                    # rows 72 bytes apart
    refused(lambda: ctx.linear_fp8(pitch, w, z(4, 32)), bad)
    off = kd.Fp8Rows(z(4 * 80 + 8, dtype=torch.uint8)[8:].view(4, 80), r.scales, 64)  # codes at 8 bytes
    refused(lambda: ctx.linear_fp8(off, w, z(4, 32)), bad)
    for call in (lambda: ctx.quantize_fp8(torch.zeros(4, 64), r),                    # host memory
                 lambda: ctx.linear_fp8(kd.Fp8Rows.empty(4, 64, device="cpu"), w, z(4, 32)),
                 lambda: ctx.linear_fp8(r, w, torch.zeros(4, 32)),
                 lambda: ctx.linear_fp8(r, w, z(4, 32), bias=torch.zeros(32)),
                 lambda: ctx.linear_fp8(r, w, z(4, 32), bias=z(31)),
                 lambda: ctx.linear_fp8(r, w, z(4, 32), bias=z(32, dtype=torch.bfloat16)),
                 lambda: ctx.rms_norm_fp8(z(4, 64), r, gain=z(128)[::2]),
                 lambda: ctx.rms_norm_fp8(z(4, 64), r, h=torch.zeros(4, 64)),
                 lambda: ctx.dequantize_fp8(r, torch.zeros(4, 64))):
        with pytest.raises(ValueError):
            call()
    ctx.linear_fp8(r, w, z(4, 32))                                                   # the context stays usable
    ctx.device_status()
