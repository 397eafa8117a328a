"""The 8-bit linear path, case by case: root-mean-square norm with the residual's addition into e4m3 rows,
rows and weights quantised and read back, and the matrix product of two such operands.

Rows in 8 bits hold e4m3 codes with one power-of-two scale (an 8-bit exponent, value 2^(byte - 127)) for each
block of 128 columns: the smallest exponent, not below -126, with max|v| <= 448 * 2^e.  A row's codes are padded
with zeros to a multiple of 128.  The exponents lie in tiles of 128 rows x 4 blocks, 512 bytes each: row r, block b
at tile (r / 128, b / 4), byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4.

With `own` false, `run` computes the operators from elementary torch operations in 32 bits; with `own` true it makes
the calls that a program makes of kd_attn.  Codes come back as the values they stand for, in bf16, which holds them
exactly (4 significant bits and a power of two).
"""
import os
import sys

import torch

own = False

BLOCK = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML_BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}  # 32 weights: an f16 scale and 32 or 16 bytes
EPS = 1e-6

_kd = _ctx = None


def _library():
    """The framework's package and this process's context on it."""
    global _kd, _ctx
    if _ctx is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kandinsky.cpp_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import kd_attn
        _kd, _ctx = kd_attn, kd_attn.Context(device=torch.cuda.current_device())
    return _kd, _ctx


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token's hidden state at the pro model's width between two layers: latency alone.
        dict(name="norm token", op="norm", rows=1, cols=4096, dtype="bf16", residual=True, gain=True),
        # The 77 text tokens of a prompt at a width that is no whole number of blocks.
        dict(name="norm text ragged", op="norm", rows=77, cols=1000, dtype="f16", residual=True, gain=True),
        # The lite video model's 31,744 tokens x 1,792, f32 hidden states as ggml keeps them, first norm of a stack.
        dict(name="norm lite video", op="norm", rows=31744, cols=1792, dtype="f32", residual=False, gain=True),
        # The pro video model's 31,744 tokens x 4,096 with the residual stream in bf16.
        dict(name="norm pro video", op="norm", rows=31744, cols=4096, dtype="bf16", residual=True, gain=True),
        # An attention output on its way to the out-projection.
        dict(name="quantize activations", op="quantize", rows=31744, cols=4096, dtype="bf16"),
        # A GGUF weight of the pro model laid out once for the product.
        dict(name="quantize q8_0 weight", op="quantize", rows=4096, cols=4096, dtype="q8_0"),
        # A few odd rows.
        dict(name="quantize few rows", op="quantize", rows=33, cols=777, dtype="f32"),
        # One conditioning vector through a wide Linear (a modulation layer): the weight's bytes are all there is.
        dict(name="linear token", op="linear", rows=1, cols=4096, out=16384, dtype="f32", bias=True),
        # A prompt's text tokens through a projection of the pro model.
        dict(name="linear text", op="linear", rows=77, cols=4096, out=4096, dtype="bf16", bias=True),
        # An odd number of tokens through the lite model's widening Linear.
        dict(name="linear lite ragged", op="linear", rows=1999, cols=1792, out=7168, dtype="f16", bias=True),
        # The pro model's out-projection over one video.
        dict(name="linear pro video", op="linear", rows=31744, cols=4096, out=4096, dtype="bf16", bias=True),
        # The pro model's widening Linear over one video: the largest product.
        dict(name="linear pro widening", op="linear", rows=31744, cols=4096, out=16384, dtype="bf16", bias=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear"])
    rows = _log_int(rng, 1, 31744)
    if op == "norm":
        return dict(op=op, rows=rows, cols=_log_int(rng, 64, 8192), dtype=rng.choice(["f32", "f16", "bf16"]),
                    residual=rng.random() < 0.7, gain=rng.random() < 0.8)
    if op == "quantize":
        dtype = rng.choice(["f32", "f16", "bf16", "q8_0", "q4_0"])
        cols = _log_int(rng, 64, 8192)
        return dict(op=op, rows=min(rows, 16384), cols=max(32, cols // 32 * 32) if dtype in GGML_BLOCK_BYTES else cols,
                    dtype=dtype)
    cols, out = _log_int(rng, 64, 4096), _log_int(rng, 64, 16384)
    return dict(op=op, rows=rows, cols=cols, out=out, dtype=rng.choice(["f32", "f16", "bf16"]),
                bias=rng.random() < 0.6)


def work(case):
    r, c = case["rows"], case["cols"]
    blocks = -(-c // BLOCK)
    if case["op"] == "linear":
        n = case["out"]
        out = r * n * DTYPES[case["dtype"]].itemsize
        return dict(bytes=(r + n) * (c + blocks) + out + (4 * n if case["bias"] else 0), flops=2.0 * r * n * c)
    if case["dtype"] in GGML_BLOCK_BYTES:
        read = r * (c // 32) * GGML_BLOCK_BYTES[case["dtype"]]
    else:
        read = r * c * DTYPES[case["dtype"]].itemsize
    held = r * (c + blocks) + 2 * r * c  # codes and exponents, and the 16-bit values read back
    if case["op"] == "quantize":
        return dict(bytes=read + held, flops=3.0 * r * c)
    # the sum is read by the next layer too: with a residual it is an output of its own
    return dict(bytes=read * (3 if case["residual"] else 1) + held + (4 * c if case["gain"] else 0), flops=8.0 * r * c)


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _hidden(g, rows, cols):
    """Hidden states: normal values, with one channel in 64 some times larger, as residual streams have them."""
    big = 1.0 + 15.0 * (torch.rand(cols, generator=g, device="cuda") < 1.0 / 64).float()
    return torch.randn(rows, cols, generator=g, device="cuda") * big


def _ggml_blocks(w, dtype):
    """Rows of ggml q8_0 / q4_0 blocks of f32 weights [rows, cols], as bytes."""
    b = w.view(w.shape[0], -1, 32)
    top = b.abs().amax(2, keepdim=True)
    d = (top / (127.0 if dtype == "q8_0" else 7.0)).half()
    q = torch.where(d > 0, b / d.float(), torch.zeros_like(b)).round()
    if dtype == "q8_0":
        codes = q.clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        n = (q.clamp(-8, 7) + 8).to(torch.uint8)
        codes = n[:, :, :16] | (n[:, :, 16:] << 4)
    return torch.cat([d.view(torch.uint8), codes], 2).reshape(w.shape[0], -1).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    r, c, op = case["rows"], case["cols"], case["op"]
    s = dict(case=case)
    if op == "linear":
        n = case["out"]
        for name, v in (("x", _hidden(g, r, c)), ("w", torch.randn(n, c, generator=g, device="cuda") / c ** 0.5)):
            codes, e = _encode(v)
            s[name] = dict(codes=codes, tiles=_tiles(e), cols=c, rows=v.shape[0])
            del v
        s["bias"] = 0.5 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["y"] = torch.empty(r, n, device="cuda", dtype=DTYPES[case["dtype"]])
        return s
    s["values"] = torch.empty(r, c, device="cuda", dtype=torch.bfloat16)
    if op == "quantize" and case["dtype"] in GGML_BLOCK_BYTES:
        s["x"] = _ggml_blocks(torch.randn(r, c, generator=g, device="cuda") / c ** 0.5, case["dtype"])
    else:
        s["x"] = _hidden(g, r, c).to(DTYPES[case["dtype"]])
    if op == "norm":
        s["residual"] = torch.randn(r, c, generator=g, device="cuda").to(s["x"].dtype) if case["residual"] else None
        s["gain"] = 1.0 + 0.1 * torch.randn(c, generator=g, device="cuda") if case["gain"] else None
        s["h"] = torch.empty_like(s["x"]) if case["residual"] else None
    return s


# ------------------------------------------------------------------ plain form
def _encode(v):
    """f32 rows [R, C] -> e4m3 codes [R, C padded to blocks] and exponent bytes [R, blocks]."""
    r, c = v.shape
    v = torch.nn.functional.pad(v, (0, -c % BLOCK)).view(r, -1, BLOCK)
    # 448 = 1.75 * 2^8: the exponent field of max|v|, one more where the significand is above 1.75
    e = (((v.abs().amax(2).view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)
    codes = (v * ((254 - e) << 23).view(torch.float32)[:, :, None]).to(torch.float8_e4m3fn)
    return codes.view(r, -1), e.to(torch.uint8)


def _decode(codes, e, cols):
    """The values of codes [R, padded] with exponent bytes [R, blocks], as f32 [R, cols]."""
    scale = (e.to(torch.int32) << 23).view(torch.float32)
    return (codes.view(e.shape[0], -1, BLOCK).float() * scale[:, :, None]).view(e.shape[0], -1)[:, :cols]


def _tiles(e):
    """Exponent bytes [R, blocks] -> their tiles, as one row of bytes."""
    r, b = e.shape
    e = torch.nn.functional.pad(e, (0, -b % 4, 0, -r % 128))
    return e.view(-1, 4, 32, e.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _untiled(tiles, rows, cols):
    blocks = -(-cols // BLOCK)
    t = tiles.view(-(-rows // 128), -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
    return t.reshape(t.shape[0] * 128, -1)[:rows, :blocks]


def _ggml_values(raw, cols, dtype):
    b = raw.view(raw.shape[0], -1, GGML_BLOCK_BYTES[dtype])
    d = b[:, :, :2].contiguous().view(torch.float16).float()
    if dtype == "q8_0":
        q = b[:, :, 2:].contiguous().view(torch.int8).float()
    else:
        q = torch.cat([b[:, :, 2:] & 15, b[:, :, 2:] >> 4], 2).float() - 8.0
    return (d * q).view(raw.shape[0], cols)


def _operand(o):
    return _decode(o["codes"], _untiled(o["tiles"], o["rows"], o["cols"]), o["cols"])


def _run_plain(s):
    case = s["case"]
    if case["op"] == "linear":
        y = _operand(s["x"]) @ _operand(s["w"]).T
        if s["bias"] is not None:
            y += s["bias"]
        return dict(y=y.to(DTYPES[case["dtype"]]))
    if case["op"] == "quantize":
        v = _ggml_values(s["x"], case["cols"], case["dtype"]) if case["dtype"] in GGML_BLOCK_BYTES else s["x"].float()
        return dict(values=_decode(*_encode(v), case["cols"]).to(torch.bfloat16))
    out = {}
    h = s["x"].float()
    if s["residual"] is not None:
        out["h"] = (h + s["residual"].float()).to(s["x"].dtype)
        h = out["h"].float()
    v = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    if s["gain"] is not None:
        v = v * s["gain"]
    out["values"] = _decode(*_encode(v), case["cols"]).to(torch.bfloat16)
    return out


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    kd, ctx = _library()
    case = s["case"]
    if case["op"] == "linear":
        x = kd.Fp8Rows(s["x"]["codes"], s["x"]["tiles"], case["cols"])
        w = kd.Fp8Rows(s["w"]["codes"], s["w"]["tiles"], case["cols"])
        return dict(y=ctx.linear_fp8(x, w, s["y"], bias=s["bias"]))
    if "rows8" not in s:  # the buffer of 8-bit rows that a program keeps beside its activations
        s["rows8"] = kd.Fp8Rows.empty(case["rows"], case["cols"])
    rows8 = s["rows8"]
    out = {}
    if case["op"] == "norm":
        ctx.rms_norm_fp8(s["x"], rows8, residual=s["residual"], gain=s["gain"], eps=EPS, h=s["h"])
        if s["h"] is not None:
            out["h"] = s["h"]
    elif case["dtype"] in GGML_BLOCK_BYTES:
        kind = kd.Q8_0 if case["dtype"] == "q8_0" else kd.Q4_0
        ctx.quantize_weight_fp8(kd.KdLinear.of(s["x"], kind, case["cols"], case["rows"]), rows8)
    else:
        ctx.quantize_fp8(s["x"], rows8)
    out["values"] = ctx.dequantize_fp8(rows8, s["values"])
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ 64 bits
def _pow2(k):
    """2^k in float64 for whole k, from the format's exponent field (exp2 may be off by an ulp, which moves ties)."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _round_blocks64(v):
    """float64 rows -> the values of their e4m3 codes under the block's power-of-two scale, from the format's
    definition: 3 fraction bits, exponents from -6, ties to even, largest 448."""
    r, c = v.shape
    v = torch.cat([v, v.new_zeros(r, -c % BLOCK)], 1).reshape(r, -1, BLOCK)
    m, k = torch.frexp(v.abs().amax(2, keepdim=True))  # max = m * 2^k, 1/2 <= m < 1; 448 = 7/8 * 2^9
    e = (k - 9 + (m > 0.875)).clamp(min=-126)
    t = v * _pow2(-e)
    step = _pow2(torch.frexp(t)[1].clamp(min=-5) - 4)
    return (torch.round(t / step) * step * _pow2(e)).reshape(r, -1)[:, :c]


def _values64(o):
    """float64 values of an operand: each column's exponent byte looked up by its row's and block's place."""
    row = torch.arange(o["rows"], device="cuda")[:, None]
    blk = torch.arange(o["cols"], device="cuda")[None, :] // BLOCK
    tile = (row // 128) * (-(-o["cols"] // (4 * BLOCK))) + blk // 4
    byte = o["tiles"][tile * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + blk % 4].to(torch.int32)
    return o["codes"][:, :o["cols"]].to(torch.float64) * _pow2(byte - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.matmul(_values64(s["x"]), _values64(s["w"]).transpose(0, 1))
        return dict(y=y if s["bias"] is None else y.add_(s["bias"].double()))
    if case["op"] == "quantize":
        if case["dtype"] in GGML_BLOCK_BYTES:
            blocks = s["x"].reshape(-1, GGML_BLOCK_BYTES[case["dtype"]])
            d = blocks[:, :2].contiguous().view(torch.float16).double()
            if case["dtype"] == "q8_0":
                v = blocks[:, 2:].contiguous().view(torch.int8).double() * d
            else:
                v = torch.cat([(blocks[:, 2:] % 16).double() - 8, (blocks[:, 2:] // 16).double() - 8], 1) * d
            return dict(values=_round_blocks64(v.reshape(case["rows"], case["cols"])))
        return dict(values=_round_blocks64(s["x"].double()))
    h = s["x"].double()
    out = {}
    if s["residual"] is not None:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()
        out["h"] = h
    v = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    out["values"] = _round_blocks64(v if s["gain"] is None else v * s["gain"].double())
    return out
