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


def token_model(p, tokens, labels, blocks, scale, masks):
    """Mean softmax cross-entropy and gradients of the residual MLP over windows of tokens
    [batch, context] in 64 bits, RMS norms.  masks: for the embeddings and each block's hidden
    activations what an element is multiplied by (1 / (1 - p) or 0)."""
    from tests import ref_mx4 as N

    eps = 1e-5
    batch, context = tokens.shape
    root = np.sqrt(p["embedding"].shape[1])
    x = embedding(p["embedding"], tokens.ravel(), root).reshape(batch, -1) * masks[0]
    z, h, a, y = [x @ p["w_in"] + p["b_in"]], [], [], []
    h.append(N.norm(z[0], "rms", eps, p["pre_0"], 0.0))
    for i in range(blocks):
        a.append(np.maximum(h[i] @ p[f"w1_{i}"] + p[f"b1_{i}"], 0) * masks[1 + i])
        y.append(a[i] @ p[f"w2_{i}"] + p[f"b2_{i}"])
        zi, hi = N.block_forward(z[i], y[i], ("rms", eps, p[f"post_{i}"], 0.0), p[f"gate_{i}"], scale,
                                 ("rms", eps, p[f"pre_{i + 1}"], 0.0))
        z.append(zi)
        h.append(hi)
    logits = h[-1] @ p["w_out"] + p["b_out"]
    e = np.exp(logits - logits.max(1, keepdims=True))
    prob = e / e.sum(1, keepdims=True)
    rows = np.arange(batch)
    loss = -np.log(prob[rows, labels]).mean()
    delta = prob.copy()
    delta[rows, labels] -= 1
    delta /= batch
    g = {"w_out": h[-1].T @ delta, "b_out": delta.sum(0, keepdims=True)}
    dh, dz = delta @ p["w_out"].T, 0.0
    for i in reversed(range(blocks)):
        b = N.block_backward(z[i + 1], y[i], ("rms", eps, p[f"post_{i}"], 0.0), p[f"gate_{i}"], scale,
                             ("rms", eps, p[f"pre_{i + 1}"], 0.0), dz, dh)
        g[f"pre_{i + 1}"], g[f"post_{i}"], g[f"gate_{i}"] = b["dgamma_pre"], b["dgamma_post"], b["dgate"].sum(0, keepdims=True)
        dz, dy = b["dr"], b["dy"]
        g[f"w2_{i}"], g[f"b2_{i}"] = a[i].T @ dy, dy.sum(0, keepdims=True)
        da = (dy @ p[f"w2_{i}"].T) * masks[1 + i] * (a[i] > 0)
        g[f"w1_{i}"], g[f"b1_{i}"] = h[i].T @ da, da.sum(0, keepdims=True)
        dh = da @ p[f"w1_{i}"].T
    b = N.block_backward(z[0], None, None, None, 1.0, ("rms", eps, p["pre_0"], 0.0), dz, dh)
    g["pre_0"] = b["dgamma_pre"]
    g["w_in"], g["b_in"] = x.T @ b["dr"], b["dr"].sum(0, keepdims=True)
    dx = (b["dr"] @ p["w_in"].T) * masks[0]
    g["embedding"] = embedding_backward(p["embedding"].shape[0], tokens.ravel(), dx.reshape(batch * context, -1), root)[0]
    return loss, g
