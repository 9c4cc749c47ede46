"""Rows at four bits (e2m1 values, one power-of-two scale per 32 elements) and their products, in float64 on the CPU:
the definitions that rag_amd.QuantizedIndex is checked against.  TEST INFRASTRUCTURE ONLY."""
import numpy as np

TABLE = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
EVEN_FIRST = np.array([0, 2, 4, 6, 1, 3, 5, 7])


def normalise(x32):
    """Rows divided by their norm as the index does it: times the power of two that brings the norm into [1/2, 1), which is exact, then
    times the rest of the factor, rounded to float32, in float32."""
    norm = np.sqrt((x32.astype(np.float64) ** 2).sum(1))
    m, e = np.frexp(np.where(norm > 0, norm, 0.5))
    inv = np.where(norm > 0, 1.0 / m, 1.0).astype(np.float32)
    return np.ldexp(x32, -e[:, None]) * inv[:, None]


def quantise(x):
    """float rows [n, dim] -> (codes uint8 [n, 16 g], scales uint8 [n, g]) in the natural layout."""
    x = np.asarray(x, dtype=np.float64)
    n, dim = x.shape
    g = (dim + 31) // 32
    p = np.zeros((n, g * 32))
    p[:, :dim] = x
    p = p.reshape(n, g, 32)
    finite = np.isfinite(p).all(2)
    p = np.where(finite[:, :, None], p, 0.0)
    a = np.abs(p).max(2)
    m, e = np.frexp(a)                                   # a = m * 2^e, m in [0.5, 1)
    s = np.where(a > 0, e - 1 - 2 + (2 * m > 1.75), -126)
    s = np.clip(s, -126, 125)
    v = np.abs(p) / np.exp2(s.astype(np.float64))[:, :, None]
    far = np.abs(v[..., None] - TABLE[EVEN_FIRST])
    code = EVEN_FIRST[far.argmin(3)]                     # the first of equally near ones: an even code
    code = code + 8 * np.signbit(p)
    code = code.reshape(n, g * 32).astype(np.uint8)
    code[:, dim:] = 0
    scales = np.where(finite, s + 127, 255).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def values(codes, scales, dim):
    """(codes, scales) -> float64 [n, dim]."""
    n, g = scales.shape
    c = np.empty((n, g * 32), dtype=np.uint8)
    c[:, 0::2] = codes & 15
    c[:, 1::2] = codes >> 4
    v = TABLE[c & 7] * np.where(c & 8, -1.0, 1.0)
    f = np.exp2(scales.astype(np.float64) - 127)
    f[scales == 255] = np.nan
    return (v.reshape(n, g, 32) * f[:, :, None]).reshape(n, g * 32)[:, :dim]


def scores(q, v):
    return np.asarray(q, np.float64) @ np.asarray(v, np.float64).T


def product_bound(q, v):
    """A bound of |computed - exact| for every score, from the definition alone: queries and values are taken as they are, a score
    is the sum of their products in fp32 in any order.  Products with a zero add nothing; the others are added with one rounding
    each, of at most half a step (2^-24) of at most the sum of |products|, and so are up to four partial sums."""
    q, v = np.abs(np.asarray(q, np.float64)), np.abs(np.asarray(v, np.float64))
    terms = (q > 0).astype(np.float64) @ (v > 0).astype(np.float64).T
    return (terms + 4) * 2.0 ** -24 * (q @ v.T)


def score_bound(q, v, digits=None):
    """A bound of |computed - exact| for every score, tighter than product_bound for long rows: per block of 128 elements eight
    roundings of half a step (2^-24) of the sum of |products|, and four for the partial sums.  Nothing is allowed for the operands,
    which enter the product whole (``digits`` once said how much of a query did, and is not used)."""
    blocks = (np.asarray(q).shape[1] + 127) // 128
    return (8 * blocks + 4) * 2.0 ** -24 * (np.abs(np.asarray(q, np.float64)) @ np.abs(np.asarray(v, np.float64)).T)
