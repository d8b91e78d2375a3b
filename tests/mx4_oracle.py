"""Microscaled 4-bit floating point in 64-bit numpy, from the definition: the oracle of the mx4 tests."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}
# e4m3: bytes 0..126 ascend, 127 is not a number
E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def nearest(value, table):
    """Index of the table's entry nearest to each value >= 0; the even index where two are as near."""
    hi = np.clip(np.searchsorted(table, value), 1, len(table) - 1)
    lo = hi - 1
    down, up = value - table[lo], table[hi] - value
    return np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))


def tensor_scale(x):
    a = np.abs(x[np.isfinite(x)])
    top = np.float32(a.max() if a.size else 0.0)
    return max(np.float32(top * np.float32(1.0 / 2688.0)), np.float32(2.0 ** -126))


def quantize(x, fmt, t=None):
    """x (rows, cols) in 64 bits -> (codes (rows, cols) 0..15, scale bytes (rows, blocks))."""
    rows, cols = x.shape
    b = BLOCK[fmt]
    blocks = -(-cols // b)
    pad = np.zeros((rows, blocks * b))
    pad[:, :cols] = x
    v = pad.reshape(rows, blocks, b)
    fine = np.isfinite(v).all(-1)
    v = np.where(fine[..., None], v, 0.0)
    top = np.abs(v).max(-1)
    if fmt == "mxfp4":
        _, e = np.frexp(top)
        power = np.where(top > 0, np.clip(e - 3, -127, 125), -127)
        scale = 2.0 ** power.astype(np.float64)
        byte = np.where(fine, power + 127, 255)
        step = scale
    else:
        byte = nearest(np.minimum(top / (6.0 * float(t)), 448.0), E4M3)
        step = E4M3[byte] * float(t)
        byte = np.where(fine, byte, 127)
    q = np.abs(v) / np.where(step > 0, step, 1.0)[..., None]
    q = np.where((step > 0)[..., None], np.minimum(q, 6.0), 0.0)
    code = nearest(q, MAGNITUDES)
    code = code + np.where(fine[..., None] & np.signbit(v), 8, 0)
    return code.reshape(rows, -1)[:, :cols].astype(np.uint8), byte.astype(np.uint8)


def scale_values(byte, fmt):
    if fmt == "mxfp4":
        return np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return np.append(E4M3, np.nan)[byte & 127]


def values(code, byte, fmt, t=None):
    v = MAGNITUDES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.repeat(scale_values(byte, fmt), BLOCK[fmt], axis=-1)[..., :code.shape[-1]]
    return v * s * (1.0 if t is None else float(t))


def pack_nibbles(code):
    if code.shape[-1] % 2:
        code = np.concatenate([code, np.zeros(code.shape[:-1] + (1,), np.uint8)], -1)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack_nibbles(byte, cols):
    return np.stack([byte & 15, byte >> 4], -1).reshape(byte.shape[:-1] + (-1,))[..., :cols]
