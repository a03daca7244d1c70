"""Block-scaled rows in numpy and 64 bits: the definition that the GPU tests
compare with, written from the formats (e4m3, e2m1, e8m0 scales per 32)."""
import numpy as np

BLOCK = 32
TOP = {8: 8, 4: 2}
HALF_BF16 = 2.0 ** -8  # half a step of bf16, relative to the value


def grid(bits):
    """Magnitudes by code."""
    mantissa, bias, n = (3, 7, 127) if bits == 8 else (1, 1, 8)
    one = 1 << mantissa
    return np.array([(c % one + (one if c >= one else 0)) / one * 2.0 ** (max(c // one, 1) - bias) for c in range(n)])


def nearest(a, bits):
    """Codes of magnitudes a >= 0 (NaN: 0): the nearest, ties to the even code, at most the largest."""
    g = grid(bits)
    middle = (g[1:] + g[:-1]) / 2
    a = np.nan_to_num(a, nan=0.0)
    at = np.searchsorted(middle, a)
    tied = a == middle[np.minimum(at, middle.size - 1)]
    return at + (tied & (at % 2 == 1))


def scale_bytes(top, bits):
    """Scale byte of blocks with the largest magnitude `top`."""
    with np.errstate(all="ignore"):
        e = np.where(top > 0, np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 1 - TOP[bits], -127)
    return np.where(np.isfinite(top), np.maximum(e, -127) + 127, 255).astype(np.uint8)


def power(byte):
    """2^(byte - 127) in 64 bits; NaN for 255."""
    b = np.asarray(byte).astype(np.int64)
    return np.where(b == 255, np.nan, np.ldexp(1.0, b - 127))


def pack(codes, bits):
    """Codes [rows, k] as stored."""
    codes = codes.astype(np.uint8)
    return codes if bits == 8 else codes[:, 0::2] | codes[:, 1::2] << 4


def unpack(stored, bits):
    if bits == 8:
        return stored
    out = np.empty((stored.shape[0], 2 * stored.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = stored & 15, stored >> 4
    return out


def quantize(x, bits):
    """x [rows, k] in 64 bits -> (stored codes, scale bytes)."""
    rows, k = x.shape
    b = x.reshape(rows, k // BLOCK, BLOCK)
    a = np.abs(b)
    top = np.where(np.isnan(a).any(-1), np.nan, np.nan_to_num(a, nan=0.0, posinf=np.inf).max(-1))
    scale = scale_bytes(top, bits)
    with np.errstate(all="ignore"):
        q = nearest(a / power(scale)[..., None], bits)
    sign = np.signbit(b).astype(np.uint8) << (bits - 1)
    codes = np.where(scale[..., None] == 255, 0, q.astype(np.uint8) | sign).reshape(rows, k)
    return pack(codes, bits), scale


def code_values(codes, bits):
    """Values of unpacked codes (e4m3's 0x7f and 0xff are NaN)."""
    low = (1 << (bits - 1)) - 1
    g = np.append(grid(bits), np.nan) if bits == 8 else grid(bits)
    v = g[codes & low]
    return np.where(codes > low, -v, v)


def values(stored, scales, bits):
    """What rows stand for, in 64 bits."""
    v = code_values(unpack(stored, bits), bits)
    return v * np.repeat(power(scales), BLOCK, 1)


def to_bf16(x):
    """Bits of x in 64 bits rounded once to bf16 (nearest, ties to even; no overflow to be rounded down)."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        e = np.maximum(np.frexp(x)[1] - 1, -126)
        step = np.ldexp(1.0, e - 7)
        y = np.rint(x / step) * step
        y = np.where(np.isfinite(x), y, x).astype(np.float32)
    bits = (y.view(np.uint32) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), 0x7FC0, bits).astype(np.uint16)


def from_bf16(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def product(a, w, a_bits):
    """(A W^T, bound of its error before the last rounding) of values in 64 bits [m, k], [n, k].

    fp32 sums: at most k + 8 additions (of a block's products, of blocks, of waves), each half a step of 2^-24 of a
    partial sum no larger than sum |a w|; truncating adders are off by a whole step: (k + 8) 2^-23 sum |a w|.
    8-bit A: of eight neighbouring products seven may lose less than 2^-13 of the largest's power of two each."""
    y = a @ w.T
    mag = np.abs(a) @ np.abs(w).T
    bound = (a.shape[1] + 8) * 2.0 ** -23 * mag
    if a_bits == 8:
        m, k = a.shape
        ga, gw = np.abs(a).reshape(m, 1, k // 8, 8), np.abs(w).reshape(1, -1, k // 8, 8)
        most = np.zeros_like(y)
        for i in range(8):
            part = slice(i * (m // 8 + 1), (i + 1) * (m // 8 + 1))
            most[part] = (ga[part] * gw).max(-1).sum(-1)
        bound = bound + 7 * 2.0 ** -13 * most
    return y, bound
