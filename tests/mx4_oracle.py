"""mx4 (microscaled 4-bit rows) from its definition, in numpy with 64 bits."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [n, d] (any float type) -> codes uint8 [n, nb, 16], scales uint8 [n, nb]."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    nb = -(-d // 32)
    v = np.zeros((n, nb * 32))
    v[:, :d] = x
    v = v.reshape(n, nb, 32)
    bad = ~np.isfinite(v).all(2)
    v = np.where(bad[:, :, None], 0.0, v)
    top = np.abs(v).max(2)
    _, e = np.frexp(top)                                       # top = m 2^e, 0.5 <= m < 1
    s = np.where(top > 0, np.maximum(e - 3, -127), -127)
    u = np.abs(np.ldexp(v, -s[:, :, None]))
    # the nearest code counts the midpoints below |element / scale|; at a midpoint the even code wins
    code = sum((u >= mid) if even else (u > mid) for mid, even in zip((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0),
                                                                      (False, True, False, True, False, True, False)))
    code = code.astype(np.uint8)
    code |= (np.signbit(v).astype(np.uint8) << 3)
    code[bad] = 0
    codes = code[:, :, 0::2] | (code[:, :, 1::2] << 4)
    scales = np.where(bad, 255, s + 127).astype(np.uint8)
    return codes, scales


def dequantize(codes, scales, d):
    """-> float64 [n, d]"""
    n, nb, _ = codes.shape
    code = np.empty((n, nb, 32), np.uint8)
    code[:, :, 0::2] = codes & 15
    code[:, :, 1::2] = codes >> 4
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = np.ldexp(v, scales.astype(np.int64)[:, :, None] - 127)
    v = np.where(scales[:, :, None] == 255, np.nan, v)
    return v.reshape(n, nb * 32)[:, :d]


def rounded(x):
    """the values of x's mx4 form, float32 (exact)"""
    return dequantize(*quantize(x), np.shape(x)[1]).astype(np.float32)
