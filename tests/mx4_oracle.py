"""MXFP4 from its definition, in numpy's 64 bits: the checker of the tabby_mx4_* operators."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def quantize(x):
    """(codes uint8 [rows, cols padded to 32], biased exponents uint8 [rows, blocks]) of a float array."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = np.zeros((rows, blocks * BLOCK))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, BLOCK)
    finite = np.isfinite(v).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(v), v, 0.0)).max(-1), 1.0)
    power = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)  # frexp's mantissa is in [1/2, 1)
    power = np.clip(power, -127, 127)
    a = np.ldexp(np.abs(np.where(finite[..., None], v, 0.0)), -power[..., None])
    code = np.zeros(a.shape, dtype=np.uint8)
    for j in range(7):
        middle = (LEVELS[j] + LEVELS[j + 1]) / 2
        code += ((a > middle) if j % 2 == 0 else (a >= middle)).astype(np.uint8)
    code |= (np.signbit(v) & finite[..., None]).astype(np.uint8) << 3
    scale = np.where(finite, power + 127, 255).astype(np.uint8)
    return code.reshape(rows, -1), scale


def values(codes, scales, cols):
    """The float64 values that codes [rows, padded] and exponents stand for."""
    rows = codes.shape[0]
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    power = scales.astype(np.int64) - 127
    v = np.ldexp(v.reshape(rows, -1, BLOCK), power[..., None])
    v = np.where((scales == 255)[..., None], np.nan, v)
    return v.reshape(rows, -1)[:, :cols]


def rounded(x):
    """The values that a float array stands for once quantised."""
    codes, scales = quantize(x)
    return values(codes, scales, np.asarray(x).shape[1])


def packed(codes):
    """Codes [rows, padded] two to a byte, the lower column in the low half."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)
