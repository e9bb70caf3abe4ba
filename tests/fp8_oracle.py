"""FP8 (e4m3) in blocks of 128 from its definition, in numpy's 64 bits: what the tabby_fp8_* operators are tested
against."""
import numpy as np

BLOCK = 128
# The 127 magnitudes: three bits of the significand, exponents from 2^-6, subnormals below.
LEVELS = np.array([m / 8 * 2.0 ** -6 for m in range(8)] +
                  [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)])[:127]
MIDDLES = (LEVELS[:-1] + LEVELS[1:]) / 2
assert LEVELS[-1] == 448.0


def decoded(codes):
    """The float64 values of e4m3 codes (127 and 255: NaN)."""
    codes = np.asarray(codes, dtype=np.uint8)
    v = np.append(LEVELS, np.nan)[codes & 127]
    return np.where(codes & 128, -v, v)


def nearest(a):
    """The index of the level nearest to each of a >= 0, an exact midpoint to the even one; a <= 448."""
    low, high = np.searchsorted(MIDDLES, a), np.searchsorted(MIDDLES, a, side="right")
    return np.where(low % 2 == 0, low, high)


def rounded(x, block_rows=1):
    """The float64 values that a float array stands for once quantised, a scale to each block_rows x 128."""
    x = np.asarray(x, dtype=np.float64)
    out = np.empty_like(x)
    for r in range(0, x.shape[0], block_rows):
        for c in range(0, x.shape[1], BLOCK):
            v = x[r:r + block_rows, c:c + BLOCK]
            if not np.isfinite(v).all():
                out[r:r + block_rows, c:c + BLOCK] = np.nan
                continue
            top = np.abs(v).max()
            power = 0
            if top > 0:
                power = int(np.frexp(top)[1]) - 9  # top in [2^(power + 8), 2^(power + 9))
                if top > np.ldexp(448.0, power):
                    power += 1
                power = max(power, -126)
            a = np.ldexp(np.abs(v), -power)
            out[r:r + block_rows, c:c + BLOCK] = np.copysign(np.ldexp(LEVELS[nearest(a)], power), v)
    return out
