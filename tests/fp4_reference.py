"""Plain 64-bit forms of the microscaled 4-bit operators (numpy): the definitions of include/vrb.h by search over the
code tables, written apart from the kernels."""
import numpy as np

NVFP4, MXFP4 = 0, 1
BLOCK = {NVFP4: 16, MXFP4: 32}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127])


def nearest(v, grid):
    """Index of the nearest grid value of every v >= 0 (ties to the even index, saturating); v on a border is exact in
    double: borders have few bits and the callers' products at most 32."""
    middle = (grid[1:] + grid[:-1]) / 2
    low, high = np.searchsorted(middle, v, side="left"), np.searchsorted(middle, v, side="right")
    return np.where(low % 2 == 0, low, high)


def row_bytes(k):
    return (k + 31) // 32 * 16


def scale_index(row, block, blocks):
    return ((row // 128) * ((blocks + 3) // 4) + block // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + block % 4


def scale_bytes(fmt, rows, k):
    blocks = -(-k // BLOCK[fmt])
    return -(-rows // 128) * -(-blocks // 4) * 512


def quantize(x, fmt, g=None):
    """x [rows, k] float -> (codes [rows, row_bytes] u8, scales u8)."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    block, blocks = BLOCK[fmt], -(-k // BLOCK[fmt])
    g = 1.0 if g is None else float(g)
    codes, scales = np.zeros((rows, row_bytes(k) * 2), np.uint8), np.zeros(scale_bytes(fmt, rows, k), np.uint8)
    for b in range(blocks):
        v = x[:, b * block:(b + 1) * block]
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            top = np.max(np.abs(v), axis=1)
            bad = ~np.isfinite(v).all(axis=1) | ~np.isfinite(g)
            top = np.where(bad, 0.0, top)
            if fmt == NVFP4:
                byte = nearest(top / (6.0 * g), E4M3) if g > 0 and np.isfinite(g) else np.zeros(rows, int)
                unit = E4M3[byte] * (g if np.isfinite(g) else 0.0)
            else:
                byte = np.where(top > 0, np.clip(np.frexp(top)[1] - 3, -127, 127) + 127, 0)
                unit = np.ldexp(1.0, byte - 127)
            ratio = np.where(unit[:, None] > 0, np.where(bad[:, None], 0.0, np.abs(v)) / np.where(unit > 0, unit, 1.0)[:, None], 0.0)
        live = (unit > 0) & ~bad & ((top > 0) | (fmt == MXFP4))
        code = (nearest(ratio, E2M1) | (np.signbit(v) << 3)) * live[:, None]
        codes[:, b * block:b * block + v.shape[1]] = code
        scales[scale_index(np.arange(rows), b, blocks)] = np.where(bad, 0x7F if fmt == NVFP4 else 0xFF, byte)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales


def parts(codes, scales, fmt, rows, k):
    """(element values, block scales) of a packed operand, both [rows, k], without the tensor scale."""
    blocks = -(-k // BLOCK[fmt])
    byte = scales[scale_index(np.arange(rows)[:, None], np.arange(blocks)[None, :], blocks)].astype(int)
    if fmt == NVFP4:
        s = np.where(byte == 127, np.nan, E4M3[np.minimum(byte, 126)])
    else:
        s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    c = np.empty((rows, codes.shape[1] * 2), np.uint8)
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    c = c[:, :k]
    return np.where(c >= 8, -1.0, 1.0) * E2M1[c & 7], np.repeat(s, BLOCK[fmt], axis=1)[:, :k]


def values(codes, scales, fmt, rows, k, g=None):
    e, s = parts(codes, scales, fmt, rows, k)
    return e * s * (1.0 if g is None else float(g))


def activation(y, kind):
    from math import erf
    if kind is None:
        return y
    with np.errstate(over="ignore"):
        if kind == 0:
            return y / (1.0 + np.exp(-y))
        if kind == 1:
            return 0.5 * y * (1.0 + np.vectorize(erf)(y / np.sqrt(2.0)))
        if kind == 2:
            return 0.5 * y * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (y + 0.044715 * y ** 3)))
        if kind == 3:
            return np.tanh(y)
        return np.maximum(y, 0.0)
