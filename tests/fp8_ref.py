"""8-bit rows in 64 bits: e4m3 codes with a power-of-two scale per 128 columns, from the format's definition.

Apart from the library's code: codes are found among the 256 values of e4m3 by nearest distance, ties to the even
code, and the scale by trying exponents against 448 * 2^e."""
import numpy as np


def e4m3_values():
    """The 256 values: sign, 4 exponent bits (bias 7), 3 fraction bits; no infinities, S.1111.111 is NaN."""
    v = np.empty(256)
    for c in range(256):
        s, e, f = -1.0 if c & 128 else 1.0, (c >> 3) & 15, c & 7
        v[c] = s * (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        if c & 127 == 127:
            v[c] = np.nan
    return v


VALUES = e4m3_values()
_POS = VALUES[:127]  # 0 .. 448, ascending with the code


def round_e4m3(t):
    """float64 values (|t| <= 448, or NaN) -> codes, to nearest, ties to the even code."""
    a = np.abs(t)
    hi = np.clip(np.searchsorted(_POS, np.where(np.isnan(a), 0, a)), 1, 126)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(a), 127, code).astype(np.uint8)
    return np.where(np.signbit(t) & ~np.isnan(a), code | 128, code).astype(np.uint8)


def encode(v):
    """float64 rows -> (codes (R, K), scale bytes (R, blocks)).  NaN and infinities take the NaN code."""
    v = np.asarray(v, np.float64)
    R, K = v.shape
    nb = -(-K // 128)
    p = np.zeros((R, nb * 128))
    p[:, :K] = np.where(np.isfinite(v), v, np.nan)
    p = p.reshape(R, nb, 128)
    top = np.nanmax(np.abs(np.nan_to_num(p, nan=0.0)), axis=2) if R else np.zeros((R, nb))
    e = np.full(top.shape, -126)
    with np.errstate(divide="ignore"):
        guess = np.where(top > 0, np.floor(np.log2(np.maximum(top, 1e-300))) - 10, -126).astype(int)
    e = np.maximum(e, guess)
    while True:  # the smallest exponent that covers the block
        low = top > 448 * 2.0 ** e
        if not low.any():
            break
        e = np.where(low, e + 1, e)
    codes = round_e4m3(p * 2.0 ** -e[:, :, None].astype(float)).reshape(R, -1)[:, :K]
    return codes, (e + 127).astype(np.uint8)


def decode(codes, scales):
    K = codes.shape[1]
    s = 2.0 ** (scales.astype(np.float64) - 127)
    return VALUES[codes] * np.repeat(s, 128, axis=1)[:, :K]


def tile_offsets(R, K):
    """Byte offset of the scale of every (row, block)."""
    nb = -(-K // 128)
    T = -(-nb // 4)
    r, b = np.arange(R)[:, None], np.arange(nb)[None, :]
    return ((r // 128) * T + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4


def round_to(v, dtype):
    """float64 -> f32 / f16 / bf16 and back, rounded once."""
    v = np.asarray(v, np.float64)
    if dtype == "f32":
        return v.astype(np.float32).astype(np.float64)
    if dtype == "f16":
        return v.astype(np.float16).astype(np.float64)
    m, k = np.frexp(v)
    return np.ldexp(np.rint(m * 256), k - 8)  # 8 significant bits (normal range)
