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


def bytes_operand(kd, codes, scales):
    """An Fp8Rows of given codes (R, K) and scale bytes (R, blocks)."""
    R, K = codes.shape
    r = kd.Fp8Rows.empty(R, K)
    c = np.zeros((R, r.codes.shape[1]), np.uint8)
    c[:, :K] = codes
    t = np.zeros(r.scales.numel(), np.uint8)
    t[fp8_ref.tile_offsets(R, K)] = scales
    r.codes.view(torch.uint8).copy_(torch.from_numpy(c))
    r.scales.copy_(torch.from_numpy(t))
    return r


def bytes_values(codes, scales):
    """What such rows are worth in float64: code * 2^(byte - 127), and NaN under the byte 255."""
    f = np.ldexp(1.0, scales.astype(int) - 127)
    f[scales == 255] = np.nan
    return fp8_ref.VALUES[codes] * np.repeat(f, 128, axis=1)[:, :codes.shape[1]]


@pytest.mark.parametrize("pad", [0, 1])
def test_read_back_of_every_scale_byte(ctx, kd, pad):
    """All 256 codes under all 256 scale bytes, into aligned rows and into rows that start anywhere."""
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 2, axis=1)
    r = bytes_operand(kd, codes, scales)
    want = torch.from_numpy(bytes_values(codes, scales)).to(torch.float32)  # exact but for what is beyond f32
    for dtype in TORCH.values():
        y = torch.empty(256, 256 + pad, device="cuda", dtype=dtype)[:, pad:]
        ctx.dequantize_fp8(r, y)
        assert torch.equal(torch.nan_to_num(y.cpu().float(), nan=12345.0), torch.nan_to_num(want.to(dtype).float(), nan=12345.0))


@pytest.mark.parametrize("M", [5, 300])
def test_product_of_the_outermost_scale_bytes(ctx, kd, M):
    """Scales of 2^-127 against 2^127 in either operand, and a block under the byte 255, which makes its row NaN."""
    K, N = 256, 130
    rng = np.random.default_rng(M)
    cx, cw = (rng.integers(0, 126, (n, K)).astype(np.uint8) | (rng.integers(0, 2, (n, K)) << 7).astype(np.uint8) for n in (M, N))
    for bx, bw in ((0, 254), (254, 0)):
        sx, sw = np.full((M, 2), bx, np.uint8), np.full((N, 2), bw, np.uint8)
        sx[3, 1] = 255
        y = torch.empty(M, N, device="cuda")
        ctx.linear_fp8(bytes_operand(kd, cx, sx), bytes_operand(kd, cw, sw), y)
        assert torch.isnan(y[3]).all() and int(torch.isnan(y).any(1).sum()) == 1
        keep = np.arange(M) != 3
        check_product(y[torch.from_numpy(keep).cuda()], bytes_values(cx, sx)[keep], bytes_values(cw, sw), None, "f32", f"{bx} {bw}")
    ctx.device_status()


@pytest.mark.parametrize("M,N,K", [(1, 16384, 4096), (5, 9600, 2100), (100, 16384, 1800), (256, 9600, 1700), (40, 9400, 4500)])
def test_few_tokens_ring_used_again(ctx, kd, M, N, K):
    """Products of few tokens whose CTAs take more blocks of 128 columns than their ring holds: stored from the sums in
    place (1 and 5 tokens), by the join of one part (100, 256) and of two (40).  K in blocks, the CTAs to a tile, and the
    ring's stages by shared memory are restated here, so that another plan cannot take the cases away unseen."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    blocks, tiles, nt = -(-K // 128), -(-N // 128), -(-M // 16) * 16
    parts = min(8, blocks, max(1, sms // tiles))
    stages = min(12, (232448 - 2048) // (128 * 128 + nt * 128 + 3 * 512))
    assert -(-blocks // parts) > stages and parts == (2 if M == 40 else 1)
    g = torch.Generator(device="cuda").manual_seed(K)
    rows = []
    for n in (M, N):
        r = kd.Fp8Rows.empty(n, K)
        c = torch.randint(0, 126, r.codes.shape, generator=g, device="cuda", dtype=torch.uint8)
        c |= torch.randint(0, 2, c.shape, generator=g, device="cuda", dtype=torch.uint8) << 7
        s = torch.randint(118, 131, (n, blocks), generator=g, device="cuda", dtype=torch.uint8)
        r.codes.view(torch.uint8).copy_(c)
        r.scales[torch.from_numpy(fp8_ref.tile_offsets(n, K)).cuda()] = s
        v = torch.from_numpy(fp8_ref.VALUES).cuda()[c[:, :K].long()]
        rows.append((r, v * torch.exp2(s.double() - 127).repeat_interleave(128, 1)[:, :K]))
    (x, x64), (w, w64) = rows
    bias = torch.randn(N, generator=g, device="cuda")
    want, room = x64 @ w64.T + bias, x64.abs() @ w64.abs().T + bias.abs()
    for name in TORCH:
        y = torch.empty(M, N, device="cuda", dtype=TORCH[name])
        ctx.linear_fp8(x, w, y, bias=bias)
        lim = HALF[name] * want.abs() + (2.0 ** -25 if name == "f16" else 0) + (K + 1) * 2.0 ** -23 * room
        big = want.abs() > 65000 if name == "f16" else torch.zeros_like(want, dtype=torch.bool)  # (beyond f16: infinite)
        assert bool((((y.double() - want).abs() <= lim) | big).all()), name
        assert torch.equal(y, ctx.linear_fp8(x, w, torch.empty_like(y), bias=bias))
    ctx.device_status()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("K,start", [(1000, 0), (1000, 1), (1537, 3), (4096, 0), (4097, 1), (5200, 0), (9000, 0), (9001, 1), (16400, 0)])
def test_norm_in_place_over_several_warps(ctx, kd, K, start, dtype):
    """The sum written over x and over the residual on rows of several warps, aligned and from odd starts, one and two
    chunks a warp, more rows than CTAs: the bits of the sum and of the rows are those of a sum written elsewhere."""
    R = 700
    g = torch.Generator(device="cuda").manual_seed(K + start)
    base = [torch.randn(R, start + K + 2, generator=g, device="cuda").to(TORCH[dtype]) for _ in range(2)]
    x, res = (t[:, start:start + K] for t in base)
    gain = 1 + 0.1 * torch.randn(K, generator=g, device="cuda")
    h, want = torch.empty_like(x), kd.Fp8Rows.empty(R, K)
    ctx.rms_norm_fp8(x, want, residual=res, gain=gain, h=h)
    assert torch.equal(h, x + res)
    for target in (0, 1):
        wide = [t.clone() for t in base]
        xi, ri = (t[:, start:start + K] for t in wide)
        r = kd.Fp8Rows.empty(R, K)
        ctx.rms_norm_fp8(xi, r, residual=ri, gain=gain, h=(xi, ri)[target])
        assert torch.equal((xi, ri)[target], h) and torch.equal((xi, ri)[1 - target], (x, res)[1 - target])
        for t, o in zip(wide, base):
            assert torch.equal(t[:, :start], o[:, :start]) and torch.equal(t[:, start + K:], o[:, start + K:])
        assert all(np.array_equal(a, b) for a, b in zip(rows_of(r), rows_of(want)))


@pytest.mark.parametrize("M", [3, 100, 300])
def test_vectors_written_by_the_call_before(ctx, kd, M):
    """A bias that the product before wrote, and a gain likewise, in one buffer over and over: the bits that the same
    calls give with a wait after each."""
    K, C = 256, 640
    w = operand(kd, hidden(C, K, 81) / np.sqrt(K))[0]
    x, x64 = operand(kd, hidden(M, K, 82))
    ones = [operand(kd, hidden(1, K, 83 + i))[0] for i in range(2)]
    rows = dev(hidden(M, C, 85), "bf16")

    def chain(sync):
        v, out = torch.zeros(C, device="cuda"), []
        for i in range(30):
            y, r = torch.empty(M, C, device="cuda"), kd.Fp8Rows.empty(M, C)
            for call in (lambda: ctx.linear_fp8(ones[i & 1], w, v), lambda: ctx.linear_fp8(x, w, y, bias=v),
                         lambda: ctx.linear_fp8(ones[1 - (i & 1)], w, v), lambda: ctx.rms_norm_fp8(rows, r, gain=v)):
                call()
                if sync:
                    torch.cuda.synchronize()
            out += [y, r.codes.view(torch.uint8)[:, :C], r.scales.clone()]
        torch.cuda.synchronize()
        return out

    fast, slow = chain(False), chain(True)
    assert all(torch.equal(a, b) for a, b in zip(fast, slow))
    assert not torch.equal(fast[0], fast[3])
    ctx.device_status()


def test_written_rows_over_each_other_are_refused(ctx, kd):
    """Tensors whose rows meet across tokens and sequences are refused as outputs; rows that interleave are written."""
    K, flat = 64, lambda n: torch.full((n,), 9.0, device="cuda")
    for N, L, sn, sl in ((3, 4, K, K), (3, 4, K, 2 * K), (2, 4, 4 * K, 2 * K), (2, 2, K, 2 * K - 1), (2, 3, 2 * K + 1, K)):
        v, r, w = flat(4096).as_strided((N, L, K), (sn, sl, 1)), kd.Fp8Rows.empty(N * L, K), kd.Fp8Rows.empty(K, K)
        x = torch.zeros(N, L, K, device="cuda")
        for call in (lambda: ctx.dequantize_fp8(r, v), lambda: ctx.rms_norm_fp8(x, r, h=v), lambda: ctx.linear_fp8(r, w, v)):
            with pytest.raises(kd.KdAttnError) as e:
                call()
            assert e.value.status == kd.ERR_INVALID_ARGUMENT and "overlap" in str(e.value)
        assert ctx.quantize_fp8(v, r) is r  # (as an input they are rows like others)
    for N, L, sn, sl in ((2, 4, K, 2 * K), (2, 4, 3 * K, 2 * K), (2, 2, 3 * K, 2 * K), (2, 2, K + 1, 2 * K + 2), (3, 2, K, 4 * K)):
        x = dev(hidden(N * L, K, 95))
        r = kd.Fp8Rows.empty(N * L, K)
        ctx.quantize_fp8(x, r)
        base = flat(4096)
        v = base.as_strided((N, L, K), (sn, sl, 1))
        ctx.dequantize_fp8(r, v)
        assert np.array_equal(f64(v.reshape(N * L, K)), fp8_ref.decode(*rows_of(r)))
        assert int((base != 9).sum()) <= N * L * K


def test_captured_beside_other_work(ctx, kd):
    """Calls that may start before the one ahead of them ends, captured behind copies, fills and elementwise kernels and
    across a fork and a join of two streams; two such graphs in turn and replayed on two streams at a time."""
    C, F = 384, 640
    w = operand(kd, hidden(F, C, 91) / np.sqrt(C))[0]
    gain = dev(1 + 0.1 * seeded((C,), 92, 0))

    def program(M):
        src = torch.empty(M, C, device="cuda", dtype=torch.bfloat16)
        x, h = torch.empty_like(src), torch.empty_like(src)
        a, b = kd.Fp8Rows.empty(M, C), kd.Fp8Rows.empty(M, C)
        y, z = torch.empty(M, F, device="cuda"), torch.empty(M, F, device="cuda")
        side = torch.cuda.Stream()

        def run():
            x.copy_(src)
            a.codes.view(torch.uint8).zero_()
            ctx.rms_norm_fp8(x, a, gain=gain, h=h)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                ctx.quantize_fp8(h, b)
                ctx.linear_fp8(b, w, z)
            ctx.linear_fp8(a, w, y)
            torch.cuda.current_stream().wait_stream(side)
            ctx.quantize_fp8(h, b)
            ctx.dequantize_fp8(b, h)
            y.add_(z)
            x.add_(h)
        return src, (x, h, y, z), run

    graphs = []
    for M, seed in ((40, 93), (300, 94)):
        src, outs, run = program(M)
        src.copy_(dev(hidden(M, C, seed), "bf16"))
        run()  # outside a graph: what each replay has to give
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append((g, src, outs, want))
    for _ in range(5):
        for g, _, outs, _ in graphs:
            for t in outs:
                t.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for _, _, outs, want in graphs for t, v in zip(outs, want))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (g, _, outs, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for _, _, outs, want in graphs for t, v in zip(outs, want))
    ctx.device_status()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("K,start", [(256, 0), (200, 1), (1024, 0), (1030, 1), (8448, 0)])
def test_norm_values_beside_the_middle_of_two_codes(ctx, kd, K, start, dtype):
    """Values within two f32 steps of the middle between two codes, on rows whose squares have an exact sum: pairs of c and
    7 c (mean 25 c^2), so the values are g / 5 and 7 g / 5, gains placing them.  Codes are those of the exact values,
    which f32 products with 1 / sqrt miss for some."""
    R = 36
    rng = np.random.default_rng(K)
    m = np.array([1.0, 7.0])[np.arange(K) % 2]
    middles = (17 + 2 * rng.integers(0, 8, K)) / 16.0 * 2.0 ** rng.integers(-2, 3, K)  # of normal codes: blocks reach 4 at least
    gain = (5 * middles / m).astype(np.float32)
    gain = (gain.view(np.int32) + rng.integers(-2, 3, K).astype(np.int32)).view(np.float32)
    c = 1 + np.arange(R)
    h = (c[:, None] * m[None, :]).astype(np.float32)
    exact = np.tile(m * gain.astype(np.float64) / 5, (R, 1))
    codes, s = fp8_ref.encode(exact)
    inv = (1 / np.sqrt(25.0 * c.astype(np.float64) ** 2)).astype(np.float32)
    in_f32 = fp8_ref.encode(((h * inv[:, None]) * gain[None, :]).astype(np.float64))[0]
    assert (in_f32 != codes).sum() >= R * K // 100
    x = torch.empty(R, start + K + 1, device="cuda", dtype=TORCH[dtype])[:, start:start + K]
    x.copy_(dev(h))
    r = kd.Fp8Rows.empty(R, K)
    ctx.rms_norm_fp8(x, r, gain=dev(gain), eps=0.0)
    got, gs = rows_of(r)
    assert np.array_equal(gs, s)
    assert np.array_equal(got, codes)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("K", [256, 1030, 9000])
def test_norm_rows_beyond_the_range_of_squares(ctx, kd, K, dtype):
    """What kd_attn.h says of rows whose squares f32 does not hold; the rows beside them are as ever."""
    x = dev(hidden(6, K, 97), dtype)
    x[0], x[2], x[4] = 0.0, 1e-24, 1e20
    for eps in (0.0, 1e-30):
        r = kd.Fp8Rows.empty(6, K)
        ctx.rms_norm_fp8(x, r, eps=eps)
        codes, s = rows_of(r)
        v = fp8_ref.VALUES[codes]
        assert np.isnan(v[[0, 2]]).all() if eps == 0 else (v[0] == 0).all() and not np.isnan(v[2]).any()
        assert (v[4] == 0).all() and (s[4] == 1).all()
        if eps:  # 1e-24 / sqrt(1e-48 + 1e-30) = 1e-9, within half an e4m3 step and f32's last bits
            got = fp8_ref.decode(codes[2:3], s[2:3])
            want = float(x[2, 0].double()) / np.sqrt(float(x[2, 0].double()) ** 2 + float(np.float32(eps)))
            assert (np.abs(got - want) <= want * (2.0 ** -4 + 2.0 ** -20)).all()
        q = kd.Fp8Rows.empty(3, K)
        ctx.rms_norm_fp8(x[1::2], q, eps=eps)
        assert np.array_equal(codes[1::2], rows_of(q)[0]) and np.array_equal(s[1::2], rows_of(q)[1])


@pytest.mark.parametrize("K", [4112, 4111])
def test_rows_past_32_bits(ctx, kd, K):
    """Buffers of more than 2^32 elements, aligned rows and odd ones: the norm with its sum, quantising, reading back and
    the product's output, looked at in the first and the last rows."""
    R, tail = (1 << 20) + 77, 70
    assert R * (K - 1) > 1 << 32
    x = torch.zeros(R, K, device="cuda", dtype=torch.bfloat16)
    ends = torch.cat([torch.arange(tail), torch.arange(R - tail, R)]).cuda()
    some = dev(hidden(2 * tail, K, 98), "bf16")
    x[ends] = some
    r, s = kd.Fp8Rows.empty(R, K), kd.Fp8Rows.empty(2 * tail, K)

    def at_ends(rows):
        off = torch.from_numpy(fp8_ref.tile_offsets(R, K)[ends.cpu().numpy()]).cuda()
        return rows.codes.view(torch.uint8)[ends, :K].cpu().numpy(), rows.scales[off].cpu().numpy()

    ctx.quantize_fp8(x, r)
    ctx.quantize_fp8(some, s)
    assert all(np.array_equal(a, b) for a, b in zip(at_ends(r), rows_of(s)))
    y = torch.full_like(x, 3.0)
    ctx.dequantize_fp8(r, y)
    assert torch.equal(y[ends], ctx.dequantize_fp8(s, torch.empty_like(some))) and not bool(y[tail:R - tail].any())
    ctx.rms_norm_fp8(x, r, residual=x, h=y)
    ctx.rms_norm_fp8(some, s, residual=some)
    assert all(np.array_equal(a, b) for a, b in zip(at_ends(r), rows_of(s)))
    assert torch.equal(y[ends], some + some) and not bool(y[tail:R - tail].any())
    a, b = kd.Fp8Rows.empty(R, 128), kd.Fp8Rows.empty(2 * tail, 128)
    few = dev(hidden(2 * tail, 128, 99))
    wide = torch.zeros(R, 128, device="cuda")
    wide[ends] = few
    ctx.quantize_fp8(wide, a)
    ctx.quantize_fp8(few, b)
    w, _ = operand(kd, hidden(K, 128, 100))
    ctx.linear_fp8(a, w, y)
    assert torch.equal(y[ends], ctx.linear_fp8(b, w, torch.empty_like(some))) and not bool(y[tail:R - tail].any())
    ctx.device_status()
