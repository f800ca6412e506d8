"""MX-FP4 in plain numpy, 64 bits, from the format's definition: what the kernels' tests compare with.

An element is an E2M1 code (magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6) times 2^(s - 127), s the E8M0 byte of its block of 32; two
codes per byte, low nibble first.  Every value is exact in 64 bits."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """(codes [m, 16 B] uint8, scales [m, B] uint8) of the rows of x (any float type, non-finite values allowed)."""
    x = np.asarray(x).astype(np.float64)
    m, k = x.shape
    blocks = np.zeros((m, -(-k // 32) * 32))
    blocks[:, :k] = x
    blocks = blocks.reshape(m, -1, 32)
    bad = ~np.isfinite(blocks).all(-1)
    safe = np.where(np.isfinite(blocks), blocks, 0.0)
    top = np.abs(safe).max(-1)
    exponent = np.frexp(np.where(top > 0, top, 1.0))[1] - 1  # floor(log2 top), exact
    s = np.where(top > 0, np.maximum(exponent - 2 + 127, 0), 0)
    a = np.abs(safe) / np.ldexp(1.0, s - 127)[..., None]
    # round to nearest, ties to the neighbour whose code is even: code i+1 begins above (i even) or at (i odd) the midpoint
    mid = (MAGNITUDES[1:] + MAGNITUDES[:-1]) / 2
    code = np.zeros(a.shape, np.uint8)
    for i, b in enumerate(mid):
        code += (a >= b) if i % 2 else (a > b)
    code |= np.where(np.signbit(safe), 8, 0).astype(np.uint8)
    code[bad] = 0
    s = np.where(bad, 255, s).astype(np.uint8)
    code = code.reshape(m, -1, 2)
    return code[..., 0] | (code[..., 1] << 4), s


def values(codes, scales, k):
    """64-bit values of packed rows, NaN where the scale byte is 255."""
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = MAGNITUDES[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    f = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * np.repeat(f, 32, -1))[..., :k]


def random_packed(g, shape, lo=110, hi=130):
    """Random codes and scales for rows of `shape` = (..., k): any code, scales in [lo, hi)."""
    *lead, k = shape
    kb = -(-k // 32)
    return (g.integers(0, 256, (*lead, 16 * kb), dtype=np.uint8), g.integers(lo, hi, (*lead, kb), dtype=np.uint8))
