"""Plain 64-bit forms of the MX4 operators, and bounds of their rounding.

EPS is half a step of fp32 (2^-24), the error of one rounding."""
import numpy as np

EPS = 2.0 ** -24
VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
# values at which the nearest code changes, and the code that a value on it takes
MIDS = (VALUES[1:] + VALUES[:-1]) / 2


def blocks(k):
    return -(-k // 32)


def quantize(x):
    """Codes [m, ceil(k / 2)] and scales [m, ceil(k / 32)] of fp32 rows."""
    m, k = x.shape
    codes = np.zeros((m, 2 * ((k + 1) // 2)), np.uint8)
    scales = np.zeros((m, blocks(k)), np.uint8)
    for j in range(blocks(k)):
        y = x[:, 32 * j:32 * j + 32].astype(np.float64)
        bad = ~np.isfinite(y).all(1)
        y = np.where(bad[:, None], 0, y)
        top = np.abs(y).max(1)
        e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127).clip(-127)
        a = np.abs(y) / 2.0 ** e[:, None]
        c = np.searchsorted(MIDS, a, side="left")           # on a midpoint: the lower code
        c += (c < 7) & (a == np.append(MIDS, 0)[np.minimum(c, 7)]) & (c % 2 == 1)  # or the even one
        c = np.where(np.signbit(y) & ~bad[:, None], c + 8, c)
        codes[:, 32 * j:32 * j + y.shape[1]] = c
        scales[:, j] = np.where(bad, 255, e + 127)
    return codes[:, ::2] | codes[:, 1::2] << 4, scales


def values(codes, scales):
    """The values of all nibbles [m, 2 * bytes] in 64 bits."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = np.where(c > 7, -VALUES[c & 7], VALUES[c & 7])
    two = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(two, 32, 1)[:, :v.shape[1]]


def codes(rng, m, kb, lo=127, hi=129):
    """Random codes of kb bytes a row with scales in lo .. hi - 1.  (With lo .. hi as they are,
    products are multiples of 1/4 below 2^8: sums of up to 2^14 of them are exact in fp32,
    in any order.)"""
    return (rng.integers(0, 256, (m, kb)).astype(np.uint8),
            rng.integers(lo, hi, (m, -(-kb // 16))).astype(np.uint8))


def product(a, sa, b, sb):
    """A B^T in 64 bits, and how far fp32 may be off: the sum of a block's products is a whole
    number of quarters below 2^13 and exact, and at most one rounding for each block and 20
    for the joining of partial sums follow, each within EPS of the sum of the sizes (and
    half of the smallest subnormal)."""
    va, vb = values(a, sa), values(b, sb)
    with np.errstate(all="ignore"):
        size = np.abs(va) @ np.abs(vb).T
        n = sa.shape[1] + 20
        return va @ vb.T, n * (EPS * size + 2.0 ** -150)


# The gate's roundings in EPS: exp(-g) is within 3 (a unit of the instruction, 2, and one of the
# correction), the divisor 1 + exp takes at most those 3 and rounds (4), its reciprocal is
# within a unit (2), and two products round: 8, and what their products add.
GATE = 9


def gated(g, tg, u, tu):
    """silu(g) * u and its bound: silu's slope is below 1.1, and the gate's own roundings.
    1 / (1 + exp(-g)) becomes 0 below g = -87.3, where silu is less than 2^-119."""
    with np.errstate(all="ignore"):
        s = g / (1 + np.exp(-g))
        out = s * u
        tol = (1.1 * tg * (np.abs(u) + tu) + np.abs(s) * tu) + GATE * EPS * np.abs(out) + 2.0 ** -119 * np.abs(u) + 2.0 ** -148
    return out, tol
