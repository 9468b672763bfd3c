"""8-bit block-scaled matrices, the embedding and dropout's mask in numpy, 64 bits: the
reference of their tests, written from the formulas."""
import numpy as np

from tests.ref_mx4 import tile_scales, untile_scales  # noqa: F401  (the 8-bit scales lie in the same order)

BLOCK = 128


def e4m3(code):
    """The value of a code s eeee mmm: subnormal for e = 0, NaN for all ones."""
    sign, e, m = -1.0 if code & 128 else 1.0, code >> 3 & 15, code & 7
    if e == 15 and m == 7:
        return np.nan
    return sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))


VALUES = np.array([e4m3(c) for c in range(256)])


def quantize(x):
    """(codes uint8 [rows, k], scale bytes uint8 [rows, blocks]) of x [rows, k]: the least
    exponent with amax <= 448 * 2^e, the nearest of the finite values, half way the even code."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    blocks = -(-k // BLOCK)
    b = np.zeros((rows, blocks * BLOCK))
    b[:, :k] = x
    b = b.reshape(rows, blocks, BLOCK)
    scales = np.zeros((rows, blocks), np.uint8)
    finite = np.isfinite(b).all(2)
    amax = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0.0)).max(2), 0.0)
    for r in range(rows):
        for j in range(blocks):
            e = -127
            while amax[r, j] > 448.0 * 2.0 ** e:
                e += 1
            scales[r, j] = e + 127 if finite[r, j] else 255
    unit = 2.0 ** (np.where(finite, scales, 127).astype(np.float64) - 127)
    a = np.where(finite[..., None], np.abs(b) / unit[..., None], 0.0)
    up = np.searchsorted(VALUES[:127], a)  # the first not below
    lo, hi = np.maximum(up - 1, 0), np.minimum(up, 126)
    dlo, dhi = a - VALUES[lo], VALUES[hi] - a
    codes = np.where((dhi < dlo) | ((dhi == dlo) & (hi % 2 == 0)), hi, lo)
    codes = (codes + np.where(np.signbit(b) & finite[..., None], 128, 0)).astype(np.uint8)
    return codes.reshape(rows, -1)[:, :k], scales


def values(codes, scales, k):
    """What (codes [rows, >= k], scales) stand for, [rows, k] float64; scale byte 255 is NaN."""
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return VALUES[codes[:, :k]] * np.repeat(s, BLOCK, 1)[:, :k]


def philox(counter, key):
    """Philox4x32 with ten rounds on whole numbers of any size: four counter words, two of key."""
    c, k = [int(v) for v in counter], [int(v) for v in key]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [q >> 32 ^ c[1] ^ k[0], q & 0xFFFFFFFF, p >> 32 ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep(rows, cols, p, seed, site=0, step=0, first_row=0):
    """(kept [rows, cols], what kept elements are divided by)."""
    bar = round(p * 65536)
    out = np.zeros((rows, -(-cols // 8) * 8), np.int64)
    for i in range(rows):
        for g in range(-(-cols // 8)):
            w = philox((g, first_row + i, step, site), (seed & 0xFFFFFFFF, seed >> 32))
            for e in range(8):
                out[i, g * 8 + e] = w[e // 2] >> 16 * (e % 2) & 0xFFFF
    return out[:, :cols] >= bar, 1.0 - bar / 65536


def embedding(table, tokens, scale):
    y = np.zeros((len(tokens), table.shape[1]))
    for i, t in enumerate(tokens):
        if t < table.shape[0]:
            y[i] = scale * table[t]
    return y


def embedding_backward(vocabulary, tokens, dy, scale):
    """(gradient, sum of the magnitudes that it sums, how many rows each token has)."""
    d, size, count = np.zeros((vocabulary, dy.shape[1])), np.zeros((vocabulary, dy.shape[1])), np.zeros(vocabulary, int)
    for i, t in enumerate(tokens):
        if t < vocabulary:
            d[t] += scale * dy[i]
            size[t] += abs(scale) * np.abs(dy[i])
            count[t] += 1
    return d, size, count
