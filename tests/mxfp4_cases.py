"""The 4-bit format in numpy, from its definition: a block of 32 values down a column shares 2^(s - 127), its
elements are one of 16.  Matrices are K x cols."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
# the element of a magnitude: how many of these it passes; at a tie (value equal to a border) the even code wins
BORDERS = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]


def up(n, m):
    return (n + m - 1) // m * m


def quantize(X):
    """(element codes, scale codes) of float64 values; K is filled up to a multiple of 32 with zeros."""
    K, cols = X.shape
    v = np.zeros((up(K, 32), cols))
    v[:K] = X
    v = v.reshape(-1, 32, cols)
    top = np.abs(v).max(axis=1)
    bad = ~np.isfinite(v).all(axis=1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(top > 0, np.frexp(np.where(bad, 1.0, top))[1] - 3, -127)
    e = np.clip(e, -127, 127)
    with np.errstate(invalid="ignore"):
        a = np.ldexp(np.abs(v), -e[:, None, :])
        code = sum(((a >= b) if tie_up else (a > b)).astype(np.uint8) for b, tie_up in BORDERS)
    code = code | (np.signbit(v).astype(np.uint8) << 3)
    return code.reshape(-1, cols), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    """float64 values of (K, cols) codes and (K / 32, cols) scales; scale 255 is NaN."""
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    power = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(power, 32, axis=0)


def pack(codes, ldq, fill=0):
    """Element bytes, column after column, ldq elements apart; what is behind the codes holds `fill`."""
    K, cols = codes.shape
    out = np.full((ldq // 2, cols), fill, dtype=np.uint8, order="F")
    out[: K // 2] = codes[0::2] | (codes[1::2] << 4)
    return out


def tile_starts(cols, offsets):
    """(first column, columns) of every row of scale tiles."""
    spans = [(0, cols)] if offsets is None else [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]
    return [(c, min(128, b - c)) for a, b in spans for c in range(a, b, 128)]


def tile(scales, offsets=None):
    """Scale bytes in tiles of 128 columns x 4 blocks, element by element from the formula."""
    blocks, cols = scales.shape
    kt = up(blocks, 4) // 4
    rows = tile_starts(cols, offsets)
    out = np.zeros((len(rows), kt, 512), dtype=np.uint8)
    for q, (c0, n) in enumerate(rows):
        for r in range(n):
            for b in range(blocks):
                out[q, b // 4, (r % 32) * 16 + (r // 32) * 4 + b % 4] = scales[b, c0 + r]
    return out.reshape(-1)


def random_operand(r, K, cols, spread=4):
    """Codes and scales of every kind (codes drawn evenly, scales within 2^+-spread); zeros behind K."""
    codes = r.integers(0, 16, (up(K, 32), cols)).astype(np.uint8)
    codes[K:] = 0
    return codes, (127 + r.integers(-spread, spread + 1, (up(K, 32) // 32, cols))).astype(np.uint8)
