"""ORACLE (test infrastructure, never a product path): microscaled E4M3 / E2M1 rows in 64-bit NumPy, from the definition.

A block is 32 columns; its scale is 2^(s - 127), the smallest in 2^-127 .. 2^127 with which the largest magnitude, rounded
to the nearest code (ties to the code whose last bit is 0, the grid continued past its end), is still a finite code.
The reference keeps its arrays in fp64 and has no counterpart: parity unpinned."""
import numpy as np

BLOCK = 32
GRID = {
    "mxfp4": np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]),
    "mxfp8": np.array([f * 2.0 ** -9 for f in range(8)]
                      + [(8 + f) * 2.0 ** (e - 3) for e in range(-6, 9) for f in range(8)][:-1]),
}
NEXT = {"mxfp4": 8.0, "mxfp8": 480.0}          # the step that would follow the largest code
FLT_EDGE = 2.0 ** 128 * (1 - 2.0 ** -25)       # from here on a number rounds past the largest float


def round_to_code(a, fmt):
    """Index of the magnitude nearest to ``a`` >= 0 on the grid continued by one step; ties to the even index."""
    grid = np.append(GRID[fmt], NEXT[fmt])
    mid = (grid[1:] + grid[:-1]) / 2
    k = np.searchsorted(mid, a, side="left")                 # a tie counts as below the middle
    tie = (k < len(mid)) & (a == mid[np.minimum(k, len(mid) - 1)])
    return k + (tie & (k % 2 == 1))


def quantise(x, fmt):
    """(codes (N, nb * 32) one per column, scales (N, nb)) of ``x`` (N, D)."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    nb = -(-d // BLOCK)
    p = np.zeros((n, nb * BLOCK))
    p[:, :d] = x
    p = p.reshape(n, nb, BLOCK)
    lost = ~(np.abs(p) < FLT_EDGE).all(-1)
    p = np.where(lost[..., None], 0.0, p)
    top = np.abs(p).max(-1)
    e = np.full(top.shape, -127)
    last = len(GRID[fmt]) - 1
    for _ in range(260):                                     # the definition, literally: one power up while it overflows
        over = round_to_code(np.ldexp(top, -e), fmt) > last
        if not over.any():
            break
        e = e + over
    q = np.ldexp(p, -e[..., None])
    codes = round_to_code(np.abs(q), fmt) + np.signbit(p) * (8 if fmt == "mxfp4" else 128)
    codes = np.where(lost[..., None], 0, codes)
    scales = np.where(lost, 255, e + 127)
    return codes.reshape(n, nb * BLOCK).astype(np.uint8), scales.astype(np.uint8)


def pack(codes, fmt):
    """The bytes of one code per column."""
    return codes if fmt == "mxfp8" else (codes[:, 0::2] + 16 * codes[:, 1::2]).astype(np.uint8)


def values(codes, scales, d, fmt):
    """The (N, D) values of one code per column."""
    sign = np.where(codes & (8 if fmt == "mxfp4" else 128), -1.0, 1.0)
    mag = np.append(GRID[fmt], np.nan)[codes & (7 if fmt == "mxfp4" else 127)]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (sign * mag * np.repeat(s, BLOCK, axis=1))[:, :d]


def store(x, fmt):
    """``x`` as it reads after quantisation."""
    x = np.asarray(x, dtype=np.float64)
    return values(*quantise(x, fmt), x.shape[1], fmt)
