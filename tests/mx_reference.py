"""The MX operators from their definitions, in 64 bits (numpy), for the tests: grids built from the element types' bits,
rounding as the nearest grid number (ties to the even code), products as float64 matrix products."""
import numpy as np

BLOCK = 32
EMAX = {"e2m1": 2, "e4m3": 8}


def grid(fmt):
    """Magnitudes by code: 8 codes of e2m1 (bias 1, one mantissa bit), 127 of e4m3 (bias 7, three; code 127 is NaN)."""
    bits, bias, count = (1, 1, 8) if fmt == "e2m1" else (3, 7, 127)
    out = []
    for c in range(count):
        e, m = c >> bits, c & ((1 << bits) - 1)
        out.append((m / 2 ** bits) * 2.0 ** (1 - bias) if e == 0 else (1 + m / 2 ** bits) * 2.0 ** (e - bias))
    return np.array(out)


def blocks(x):
    """x (..., k) with zeros up to whole blocks, as (..., blocks, 32) float64."""
    x = np.asarray(x, dtype=np.float64)
    pad = -x.shape[-1] % BLOCK
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (pad,))], -1)
    return x.reshape(x.shape[:-1] + (-1, BLOCK))


def quantize(x, fmt, rule="floor"):
    """(codes one per element as uint8 (..., k), scale bytes (..., blocks)) of x along its last axis."""
    k = np.asarray(x).shape[-1]
    b = blocks(x)
    g = grid(fmt)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(top)
    safe = np.where(bad | (top == 0), 1.0, top)
    mant, ex = np.frexp(safe)                                    # safe = mant 2^ex, mant in [1/2, 1)
    e = ex - 1 - EMAX[fmt]
    if rule == "ceil":
        e = e + (mant * 2 * 2.0 ** EMAX[fmt] > g[-1])
    s = np.where(top == 0, 0, np.clip(e + 127, 0, 254))
    v = np.abs(np.where(bad[..., None], 0.0, b)) * 2.0 ** (127.0 - s[..., None])
    mid = (g[1:] + g[:-1]) / 2
    lo, hi = np.searchsorted(mid, v, side="left"), np.searchsorted(mid, v, side="right")
    code = np.where(lo % 2 == 0, lo, hi)
    code = code + np.signbit(b) * (8 if fmt == "e2m1" else 128)
    code = np.where(bad[..., None], 7 if fmt == "e2m1" else 127, code)
    s = np.where(bad, 255, s)
    return code.reshape(code.shape[:-2] + (-1,))[..., :k].astype(np.uint8), s.astype(np.uint8)


def decode(codes, scales, fmt):
    """The numbers (float64) that codes (one per element) and scale bytes stand for."""
    g = grid(fmt)
    sign = 8 if fmt == "e2m1" else 128
    mag = np.concatenate([g, [np.nan]]) if fmt == "e4m3" else g
    v = mag[codes % sign] * np.where(codes >= sign, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(s, BLOCK, -1)[..., :codes.shape[-1]]


def rounded(x, fmt, rule="floor"):
    return decode(*quantize(x, fmt, rule), fmt)


def pack(codes, fmt):
    """One code per element to the stored bytes (e2m1: two a byte, the even one in the lower half)."""
    if fmt == "e4m3":
        return codes
    if codes.shape[-1] % 2:
        codes = np.concatenate([codes, np.zeros(codes.shape[:-1] + (1,), np.uint8)], -1)
    return codes[..., 0::2] | (codes[..., 1::2] << 4)
