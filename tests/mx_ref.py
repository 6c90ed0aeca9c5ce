"""Microscaled blocks in plain numpy, from the definition (include/tmt_mx.h): what the tests compare the kernels with."""
import numpy as np

MAXV = {"e2m1": 6.0, "e4m3": 448.0, "e5m2": 57344.0}


def grid(fmt):
    """Non-negative values of an element type in the order of their codes."""
    ebits, mbits, top = {"e2m1": (2, 1, 7), "e4m3": (4, 3, 0x7e), "e5m2": (5, 2, 0x7b)}[fmt]
    bias = (1 << (ebits - 1)) - 1
    out = []
    for code in range(top + 1):
        e, m = code >> mbits, code & ((1 << mbits) - 1)
        out.append(m * 2.0 ** (1 - bias - mbits) if e == 0 else (1 + m / (1 << mbits)) * 2.0 ** (e - bias))
    return np.array(out)


def quantize(x, fmt):
    """x (rows, cols) float64 -> (codes uint8 one per element, scale bytes uint8 (rows, cols / 32))."""
    rows, cols = x.shape
    b = np.asarray(x, np.float64).reshape(rows, cols // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    safe = np.where(bad[..., None], 0.0, b)
    amax = np.abs(safe).max(-1)
    e = np.full(amax.shape, -127)
    while True:                                        # the smallest exponent at which nothing passes the largest value
        over = amax > MAXV[fmt] * 2.0 ** e
        if not over.any():
            break
        e = e + over
    a = np.abs(safe) / 2.0 ** e[..., None].astype(np.float64)
    vals = grid(fmt)
    mid = (vals[1:] + vals[:-1]) / 2
    low, high = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
    code = np.where(low % 2 == 0, low, high)           # they differ on a midpoint alone: the even code
    sign = {"e2m1": 8, "e4m3": 128, "e5m2": 128}[fmt]
    code = code + sign * np.signbit(safe)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(rows, cols).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, fmt):
    """float64 values of one code per element and row-major scale bytes."""
    rows, cols = codes.shape
    sign = {"e2m1": 8, "e4m3": 128, "e5m2": 128}[fmt]
    v = grid(fmt)[codes % sign] * np.where(codes >= sign, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(rows, -1, 32) * s[..., None]).reshape(rows, cols)


def q(x, fmt):
    return values(*quantize(x, fmt), fmt)


def pack4(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack4(packed):
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = packed & 15, packed >> 4
    return out


def tile_index(rows, blocks):
    """Index of every scale byte of a 4-bit matrix in its tiles."""
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return ((r // 128) * ((blocks + 3) // 4) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def tile(scales, fill=0):
    rows, blocks = scales.shape
    out = np.full((rows + 127) // 128 * ((blocks + 3) // 4) * 512, fill, np.uint8)
    out[tile_index(rows, blocks)] = scales
    return out
