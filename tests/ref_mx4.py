"""Microscaled 4-bit matrices and the residual-block norms in numpy, 64 bits:
the reference of their tests, written from the formulas."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(codes uint8 [rows, 32 * blocks], scale bytes uint8 [rows, blocks]) of
    x [rows, k]: exponent floor(log2 amax) - 2, the nearest of the eight
    magnitudes, half way the even code."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    blocks = -(-k // 32)
    b = np.zeros((rows, blocks * 32))
    b[:, :k] = x
    b = b.reshape(rows, blocks, 32)
    codes = np.zeros(b.shape, np.uint8)
    scales = np.zeros((rows, blocks), np.uint8)
    for r in range(rows):
        for j in range(blocks):
            v = b[r, j]
            if not np.all(np.isfinite(v)):
                scales[r, j] = 255
                continue
            amax = np.abs(v).max()
            e = -127 if amax == 0 else max(int(np.frexp(amax)[1]) - 1 - 2, -127)
            scales[r, j] = e + 127
            a = np.abs(v) / 2.0 ** e
            dist = np.abs(a[:, None] - MAGNITUDES[None, :])
            near = dist.min(1, keepdims=True)
            for i in range(32):
                best = np.flatnonzero(dist[i] == near[i])
                even = [c for c in best if c % 2 == 0]
                codes[r, j, i] = (even or list(best))[0] + (8 if np.signbit(v[i]) else 0)
    return codes.reshape(rows, -1), scales


def values(codes, scales, k):
    """What (codes, scales) stand for, [rows, k] float64; scale byte 255 is NaN."""
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(codes.shape[0], -1, 32) * s[:, :, None]).reshape(codes.shape[0], -1)[:, :k]


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def tile_scales(scales, fill=0):
    """Row-major scale bytes to the device order; `fill` in the rows that only pad."""
    rows, blocks = scales.shape
    tiles, groups = -(-rows // 128), -(-blocks // 4)
    out = np.zeros((tiles * 128, groups * 4), np.uint8)
    out[rows:] = fill
    out[:rows, :blocks] = scales
    return np.ascontiguousarray(out.reshape(tiles, 4, 32, groups, 4).transpose(0, 3, 2, 1, 4))


def untile_scales(tiled, rows, blocks):
    tiles, groups = -(-rows // 128), -(-blocks // 4)
    t = np.asarray(tiled, np.uint8).reshape(tiles, groups, 32, 4, 4).transpose(0, 3, 2, 1, 4)
    return t.reshape(tiles * 128, groups * 4)[:rows, :blocks]


def _stat(x, kind, eps):
    if kind == "none":
        return np.zeros((x.shape[0], 1)), np.ones((x.shape[0], 1))
    mu = x.mean(1, keepdims=True) if kind == "layer" else np.zeros((x.shape[0], 1))
    return mu, 1.0 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + eps)


def norm(x, kind, eps, gamma, beta):
    mu, rho = _stat(x, kind, eps)
    return (x - mu) * rho * gamma + beta


def block_forward(r, y, post, gate, scale, pre):
    """(z, h); post and pre are (kind, eps, gamma, beta), y None for no block."""
    z = r if y is None else r + scale * gate * norm(y, *post)
    return z, norm(z, *pre)


def _norm_back(x, kind, eps, gamma, d):
    mu, rho = _stat(x, kind, eps)
    hat = (x - mu) * rho
    a = d * gamma
    if kind == "none":
        return a, (d * hat).sum(0, keepdims=True), d.sum(0, keepdims=True)
    dx = a - hat * (a * hat).mean(1, keepdims=True)
    if kind == "layer":
        dx -= a.mean(1, keepdims=True)
    return dx * rho, (d * hat).sum(0, keepdims=True), d.sum(0, keepdims=True)


def block_backward(z, y, post, gate, scale, pre, dz, dh):
    """Gradients by name; dgate before it is reduced to the gate's shape."""
    out = {}
    back, out["dgamma_pre"], out["dbeta_pre"] = _norm_back(z, *pre[:3], dh)
    out["dr"] = dz + back
    if y is not None:
        dt = scale * out["dr"]
        out["dgate"] = dt * norm(y, *post)
        out["dy"], out["dgamma_post"], out["dbeta_post"] = _norm_back(y, *post[:3], dt * gate)
    return out
