"""Microscaled 4-bit (MXFP4) operators restated in float64 on the CPU, element by element from the format's definition:
blocks of 32 values, scale 2^(s - 127) with s = max(E - 2, 0) (E = biased fp32 exponent of the largest magnitude), codes
0 .5 1 1.5 2 3 4 6 rounded to nearest with ties to the even code, saturated; a block with a NaN or infinity is NaN."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SIGNED = np.concatenate([LEVELS, -LEVELS])


def quantize(x):
    """x [M,K] (float64 values of a 32- or 16-bit type) -> (codes [M, 64*ceil(K/128)], scales [M, 4*ceil(K/128)]) uint8."""
    x = np.asarray(x, dtype=np.float64)
    M, K = x.shape
    Kp = -(-K // 128) * 128
    v = np.zeros((M, Kp))
    v[:, :K] = x
    v = v.reshape(M, Kp // 32, 32)
    bad = ~np.isfinite(v).all(axis=2)
    v = np.where(bad[:, :, None], 0.0, v)
    amax = np.abs(v).max(axis=2)
    _, e = np.frexp(amax)                          # amax = m * 2^e, m in [0.5, 1): floor(log2) = e - 1
    E = np.where(amax < 2.0 ** -126, 0, e - 1 + 127)
    s = np.maximum(E - 2, 0)
    a = np.abs(np.ldexp(v, (127 - s)[:, :, None]))
    dist = np.abs(a[..., None] - LEVELS)           # nearest level; of two at the same distance the even code
    best = dist.min(axis=-1, keepdims=True)
    near = dist == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + 8 * np.signbit(v)
    s = np.where(bad, 255, s)
    code = np.where(bad[:, :, None], 0, code).reshape(M, Kp).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), s.astype(np.uint8)


def dequantize(codes, scales, K):
    """float64 values [M,K] of packed rows."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)
    v = np.ldexp(SIGNED[c].reshape(c.shape[0], -1, 32), scales.astype(np.int64)[:, :, None] - 127)
    v = np.where(scales[:, :, None] == 255, np.nan, v)
    return v.reshape(c.shape[0], -1)[:, :K]


def rounded(x):
    """The values that the rows' codes stand for."""
    return dequantize(*quantize(x), np.asarray(x).shape[1])


def activation(act, z, pre, post):
    """(post * f(pre z), its derivative with respect to z)."""
    t = pre * z
    if act == "none":
        return post * t, np.full_like(z, post * pre)
    if act == "relu":
        return post * np.where(t <= 0, 0.0, t), post * pre * (t > 0)
    if act == "sin":
        return post * np.sin(t), post * pre * np.cos(t)
    s = 1.0 / (1.0 + np.exp(-t))
    return post * s, post * pre * s * (1.0 / (1.0 + np.exp(t)))


def linear(xq, wq, b, act="none", pre=1.0, post=1.0):
    """(y, dy/dz, z) from rounded operands."""
    z = xq @ wq.T + (0.0 if b is None else np.asarray(b, dtype=np.float64))
    return (*activation(act, z, pre, post), z)


def linear_backward(dy, slope, xq, wq):
    """(dx, dW, db)."""
    dz = np.asarray(dy, dtype=np.float64) * slope
    return dz @ wq, dz.T @ xq, dz.sum(axis=0)
